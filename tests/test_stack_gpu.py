"""GDN layers on a residual stream (stack.py)."""

import pytest
import torch

from gdn_18646_amd.gdn_layer import GDNLayerCustom, make_weights
from gdn_18646_amd.stack import GDNStack
from tests.helpers import assert_out_close

pytestmark = pytest.mark.gpu

D, H, DK, DV = 256, 2, 128, 128


@pytest.fixture(scope="module")
def layers(dev):
    g = torch.Generator().manual_seed(0)
    out = []
    for _ in range(3):
        w = make_weights(dev, D=D, H=H, DK=DK, DV=DV, generator=g)
        w["norm_gamma"] = (1 + 0.1 * torch.randn(D, generator=g)).to(torch.bfloat16).to(dev)
        out.append(GDNLayerCustom(w))
    return out


def _x(shape, dev, seed=1):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(dev)


def test_layer_takes_a_normed_input(layers, dev):
    x = _x((2, 70, D), dev)
    for kw in ({}, dict(return_state=True), dict(cu_seqlens=[0, 30, 70])):
        xx = x[:1] if "cu_seqlens" in kw else x
        xn = layers[0]._rmsnorm(xx.reshape(-1, D)).reshape(xx.shape)
        a, b = layers[0].forward(xx, **kw), layers[0].forward(None, xn=xn, **kw)
        if kw.get("return_state"):
            assert torch.equal(a[0], b[0]) and all(torch.equal(a[1][k], b[1][k]) for k in a[1])
        else:
            assert torch.equal(a, b)


@pytest.mark.parametrize("B,T", [(1, 3), (1, 20), (2, 3), (2, 20), (1, 2)])
def test_a_state_does_not_share_the_normed_input(layers, dev, B, T):
    """Decoding in place from the state of a forward call leaves the call's xn as it was."""
    x = _x((B, T, D), dev, 8)
    xn = layers[0]._rmsnorm(x.reshape(-1, D)).reshape(B, T, D)
    keep = xn.clone()
    _, state = layers[0].forward(None, xn=xn, return_state=True)
    _, want = layers[0].forward(x, return_state=True)
    for t in range(3):
        y, _ = layers[0].decode(_x((B, 1, D), dev, 30 + t), state, inplace=True)
        y2, _ = layers[0].decode(_x((B, 1, D), dev, 30 + t), want, inplace=True)
        assert torch.equal(y, y2)
    assert torch.equal(xn, keep)
    assert all(torch.equal(state[k], want[k]) for k in want)


@pytest.mark.parametrize("post,scaled,final", [(False, False, True), (True, True, True), (True, False, False)])
def test_stack_is_its_layers(layers, dev, post, scaled, final):
    """Against the same chain written out in fp32 torch around the layers; each of
    the three joins rounds where the chain does, and their inputs differ by the
    norm's rounding alone (the layer's own parity bar covers what it makes of it)."""
    x = _x((2, 70, D), dev)
    pg = [_x((D,), dev, 5 + i) if post else None for i in range(3)]
    sc = [_x((D,), dev, 9 + i) if scaled else None for i in range(3)]
    fg = _x((D,), dev, 20) if final else None
    stack = GDNStack(layers, fg, pg, sc, residual_scale=0.5)
    got = stack.forward(x)

    def norm(t, g):
        t = t.float()
        return t * (t.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt() * g.float()

    h = x
    for i, layer in enumerate(layers):
        y = layer.forward(h)
        u = norm(y, pg[i]) if post else y.float()
        h = (h.float() + 0.5 * (sc[i].float() if scaled else 1.0) * u).to(torch.bfloat16)
    assert_out_close(got, norm(h, fg).to(torch.bfloat16) if final else h)


def test_prefill_then_decode(layers, dev):
    """A token decoded after a prefill is the prefill's last one of a longer prompt."""
    x = _x((2, 40, D), dev, 3)
    stack = GDNStack(layers, _x((D,), dev, 4))
    want = stack.forward(x)
    out, states = stack.forward(x[:, :39], return_state=True)
    y, new = stack.decode(x[:, 39:], states)
    assert_out_close(out, want[:, :39])
    assert_out_close(y, want[:, 39:])
    y2, same = stack.decode(x[:, 39:], states, inplace=True)
    assert same is states and torch.equal(y2, y)
    assert all(torch.equal(a[k], b[k]) for a, b in zip(new, states) for k in a)


def test_packed_sequences(layers, dev):
    x = _x((1, 75, D), dev, 6)
    stack = GDNStack(layers, _x((D,), dev, 7))
    got = stack.forward(x, cu_seqlens=[0, 20, 20, 75])
    assert_out_close(got[:, :20], stack.forward(x[:, :20]))
    assert_out_close(got[:, 20:], stack.forward(x[:, 20:]))


def test_refusals(layers, dev):
    with pytest.raises(ValueError, match="needs a layer"):
        GDNStack([])
    with pytest.raises(ValueError, match="post_gammas"):
        GDNStack(layers, post_gammas=[None])
    stack = GDNStack(layers)
    states = stack.init_decode_state(1)
    x = _x((1, 1, D), dev)
    for call in (lambda s: stack.decode(x, s, inplace=True), lambda s: stack.forward(x, states=s)):
        with pytest.raises(ValueError, match="2 states"):
            call(states[:2])
    with pytest.raises(ValueError, match="state for each layer"):
        stack.decode(x, None)
    assert all((t == 0).all() for s in states for t in s.values())
