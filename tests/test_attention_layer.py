"""layers.SelfAttention with heads, learned positions and the recomputing form, alone and inside the networks and
trainers."""
import pytest
import torch

from helpers import rel


def _layer64(layer, x, heads):
    import torch.nn.functional as F
    w = {k: getattr(layer, k).conv.conv.weight.detach().double() for k in ("query_conv", "key_conv", "value_conv", "final_conv")}
    q, k, v = F.conv1d(x, w["query_conv"]), F.max_pool1d(F.conv1d(x, w["key_conv"]), 4), F.max_pool1d(F.conv1d(x, w["value_conv"]), 4)
    B, T, Tk = x.shape[0], x.shape[2], k.shape[2]
    s = torch.matmul(k.view(B, heads, -1, Tk).transpose(2, 3), q.view(B, heads, -1, T))
    if layer.positions is not None:
        b = layer.buckets
        where = torch.tensor([[b.bucket(4 * i + 2 - t) for t in range(T)] for i in range(Tk)])
        s = s + layer.positions.detach().double()[where].permute(2, 0, 1)
    p = torch.softmax(s, 2)
    mixed = torch.matmul(v.view(B, heads, -1, Tk), p).reshape(B, -1, T)
    return 0.9 * F.conv1d(mixed, w["final_conv"]) + x, p


@pytest.mark.gpu
@pytest.mark.parametrize("C,T,B,heads,buckets", [(64, 512, 3, 1, 0), (256, 32, 4, 4, 0), (64, 256, 2, 2, 16), (128, 132, 2, 1, 32)])
def test_layer_in_both_forms(dev, C, T, B, heads, buckets):
    """Output, map, gradients of input and parameters, and the gradient of a gradient penalty: the stored form against
    float64 (the existing layer test's bound), the recomputing form against it."""
    from eeggan_amd import ops
    from eeggan_amd.layers import SelfAttention
    torch.manual_seed(C + T)
    layer = SelfAttention(C, False, "kaiming_normal", heads=heads, buckets=buckets, max_distance=100)
    with torch.no_grad():
        layer.gamma.fill_(0.9)
        if buckets:
            layer.positions.normal_()
    x = torch.randn(B, C, T)
    want, p = _layer64(layer, x.double(), heads)
    layer = layer.to(dev)
    res = {}
    cot = torch.randn(B, C, T).to(dev)
    for mode in ("stored", "recompute"):
        before = ops.set_attention(mode)
        try:
            xg = x.to(dev).requires_grad_(True)
            out, amap = layer(xg)
            params = [q for q in layer.parameters()]
            first = torch.autograd.grad(out, [xg] + params, cot, create_graph=True)
            second = torch.autograd.grad((first[0] ** 2).sum(), [xg] + params)
            plain = torch.autograd.grad(layer(xg)[0], [xg] + params, cot)
        finally:
            ops.set_attention(before)
        assert rel(out, want) < 1e-5
        if mode == "stored":
            assert rel(amap.reshape(p.shape), p) < 1e-5
        else:
            assert amap is None
        res[mode] = (first, second, plain)
    for a, b in zip(res["stored"], res["recompute"]):
        for x1, x2 in zip(a, b):
            assert rel(x2, x1) < 5e-5, (x1.shape, rel(x2, x1))


@pytest.mark.gpu
@pytest.mark.parametrize("options", [dict(), dict(heads=2, buckets=16, max_distance=64)], ids=["plain", "heads+positions"])
def test_trainers_with_recomputed_attention(dev, options):
    """A whole training step (penalty included) with the recomputing form follows the stored form, eager and captured."""
    import test_e2e_gpu as E
    from eeggan_amd import layers, ops
    from eeggan_amd.graphs import GraphedTrainer
    from eeggan_amd.trainer import Trainer

    def prepare(g, d):
        with torch.no_grad():
            g.dummy[0].gamma.fill_(0.5)
            d.dummy[0].gamma.fill_(-0.5)
            gen = torch.Generator().manual_seed(3)
            for net in (g, d):
                if net.dummy[0].positions is not None:
                    net.dummy[0].positions.copy_(torch.randn(net.dummy[0].positions.shape, generator=gen))

    kw = dict(models=dict(shared=dict(self_attention_layers=[0], attention_options=options)), prepare=prepare)
    layers.set_drop_mode("device")
    try:
        base = E._two_steps(dev, Trainer, lr=0.0, **kw)
        ops.set_attention("recompute")
        eager = E._two_steps(dev, Trainer, lr=0.0, **kw), E._two_steps(dev, Trainer, **kw)
        graphed = E._two_steps(dev, GraphedTrainer, lr=0.0, **kw), E._two_steps(dev, GraphedTrainer, **kw)
    finally:
        ops.set_attention("stored")
        layers.set_drop_mode("numpy")
    # The two forms round the layer's output differently (~1e-7), so among the millions of pre-activations that follow one
    # within that of zero changes its LeakyReLU branch: it replaces one of the summands of a weight's gradient, of which
    # there are at least batch x length = 8 x 32 = 256, i.e. up to 2 / 256 of the scale with both branches' summands.  With
    # lr = 0 the moments of all iterations are compared; a step with beta1 = 0 moves an element by its gradient's SIGN, so
    # displacements of forms that round every element differently say nothing.  The captured form runs the eager form's
    # kernels: the level of the attention layer's graph test, displacements included.
    for k, a in base.items():
        if k.endswith((".m", ".v")):
            assert float((a - eager[0][k]).abs().max()) <= 2.0 / 256 * float(a.abs().max()), k
        else:
            assert torch.equal(a, eager[0][k]), k
    E._same_trajectory(eager, graphed, "recomputed attention, captured", moment_tol=5e-5)


def test_default_layer_keeps_its_parameters():
    """No option set: the reference's state dict and the same draws; positions start at zero and draw nothing."""
    from eeggan_amd import ops
    from eeggan_amd.layers import SelfAttention
    torch.manual_seed(1)
    a = SelfAttention(64, False, "kaiming_normal")
    torch.manual_seed(1)
    b = SelfAttention(64, False, "kaiming_normal", heads=4, buckets=16)
    assert "positions" not in a.state_dict() and b.state_dict()["positions"].shape == (16, 4)
    assert not b.positions.any()
    for k, v in a.state_dict().items():
        assert torch.equal(v, b.state_dict()[k])
    with pytest.raises(ValueError):
        SelfAttention(64, False, heads=3)
    assert ops.get_attention() == "stored"


def test_networks_take_attention_options():
    from eeggan_amd import config
    g, d = config.build_models(5, shared=dict(self_attention_layers=[0, 3], attention_options=dict(heads=2, buckets=8)))
    for net in (g, d):
        assert [m.heads for m in net.dummy] == [2, 2] and "dummy.1.positions" in net.state_dict()
