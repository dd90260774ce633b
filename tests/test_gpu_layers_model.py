"""GPU tests of the drop-in conditional VAE on the layer operators (layer_kernels=True): same values and
gradients as its torch layers, the operators' own composition with 8-bit checkpoints, and the state that a
training step leaves behind."""
import importlib
import sys

import pytest
import torch

import afiv_bootstrap

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def vae():
    for p in afiv_bootstrap.dropin_paths():
        if p not in sys.path:
            sys.path.insert(0, p)
    return importlib.import_module("cvae_model").ConditionalVAE_SingleHeston


def pair(vae, seed=0, **kw):
    """(model on torch layers, model on the layer operators), same weights."""
    torch.manual_seed(seed)
    a = vae(dropout=kw.pop("dropout", 0.0), **{k: v for k, v in kw.items() if k != "checkpoint8"}).cuda()
    b = vae(dropout=a.dropout, layer_kernels=True, **kw).cuda()
    b.load_state_dict(a.state_dict())
    return a, b


def batch(m, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(m, 5, generator=g, device="cuda"), torch.randn(m, 8, generator=g, device="cuda"), torch.randn(m, 4, generator=g, device="cuda"))


def near(a, b, what):
    """Two FP32 evaluations of the same few layers: sums of up to 128 products and a dozen roundings each, on values of order 1;
    batch statistics amplify by 1 / sqrt(var), of order 10 here."""
    assert torch.allclose(a, b, rtol=2e-3, atol=2e-4 * max(1.0, float(b.abs().max()))), (what, float((a - b).abs().max()))


@pytest.mark.parametrize("acts", [("tanh", "relu"), ("leaky_relu", "tanh")])
@pytest.mark.parametrize("m", [2, 64, 3000])
def test_training_step_matches_the_torch_layers(vae, m, acts):
    a, b = pair(vae, encoder_activation=acts[0], decoder_activation=acts[1])
    x, c, z = batch(m)
    da = a.double()
    for model, dt in ((da, torch.float64), (b, torch.float32)):
        model.train()
        mu, logvar = model.encode(x.to(dt), c.to(dt))
        y = model.decode(z.to(dt), c.to(dt))
        (mu.square().mean() + logvar.mean() + y.square().mean()).backward()
        model.out = (mu, logvar, y)
    if m > 2:                                             # two rows normalise to +-1: their gradients cancel to rounding
        for u, v, what in zip(b.out, da.out, ("mu", "logvar", "decode")):
            near(u.detach(), v.detach().float(), what)
        for (name, p), q in zip(b.named_parameters(), da.parameters()):
            near(p.grad, q.grad.float(), name)
    for (name, u), v in zip(b.named_buffers(), da.buffers()):
        if "num_batches" in name:
            assert int(u) == int(v) == 1
        else:
            near(u, v.float(), name)
    assert all(torch.isfinite(p.grad).all() for p in b.parameters())


def test_frozen_statistics_and_inference(vae):
    a, b = pair(vae)
    x, c, z = batch(500)
    for model in (a, b):
        model.train()
        with torch.no_grad():
            model.encode(3 * x + 1, c)
        torch.manual_seed(5)
        model.decoder(torch.cat([z, c], dim=1))           # moves the decoder's statistics
    b.load_state_dict(a.state_dict())
    a.eval(), b.eval()
    with torch.no_grad():
        for u, v in zip(b.encode(x, c), a.encode(x, c)):
            near(u, v, "encode")
        assert torch.equal(b.decode(z, c), a.decode(z, c))       # both the decoder kernel
    y, w = b.decode(z, c), a.decode(z, c)
    near(y.detach(), w.detach(), "decode with a graph")
    y.square().mean().backward()
    w.square().mean().backward()
    for (name, p), q in zip(b.named_parameters(), a.parameters()):
        if name.startswith("decoder"):
            near(p.grad, q.grad, name)


def test_checkpointed_step_is_the_operators_composition(vae):
    afiv = afiv_bootstrap.load()
    _, b = pair(vae, dropout=0.15, checkpoint8=True)
    x, c, _ = batch(200)
    b.train()
    torch.manual_seed(11)
    mu, _ = b.encode(x, c)
    mu.backward(torch.ones_like(mu))
    torch.manual_seed(11)
    h, tape = torch.cat([x, c], dim=1), []
    mods = list(b.encoder)
    for i in range(0, len(mods), 4):
        lin, bn = mods[i], mods[i + 1]
        t, s1 = afiv.linear_act_forward(h, lin.weight, lin.bias, checkpoint8=True)
        keep = torch.rand(t.shape, device="cuda") >= 0.15
        h, s2 = afiv.batch_norm_act_forward(t, bn.weight, bn.bias, act="tanh", keep=keep, drop_p=0.15, checkpoint8=True)
        assert s1.x is None and s2.x is None              # nothing but codes is kept
        tape.append((lin, bn, s1, s2))
    y, s = afiv.linear_act_forward(h, b.fc_mu.weight, b.fc_mu.bias, checkpoint8=True)
    assert torch.equal(y, mu.detach())
    g, dw, db = afiv.linear_act_backward(torch.ones_like(y), b.fc_mu.weight, s)
    assert torch.equal(dw, b.fc_mu.weight.grad) and torch.equal(db, b.fc_mu.bias.grad)
    for lin, bn, s1, s2 in reversed(tape):
        g, dgamma, dbeta = afiv.batch_norm_act_backward(g, bn.weight, bn.bias, s2)
        assert torch.equal(dgamma, bn.weight.grad) and torch.equal(dbeta, bn.bias.grad)
        g, dw, db = afiv.linear_act_backward(g, lin.weight, s1)
        assert torch.equal(dw, lin.weight.grad) and torch.equal(db, lin.bias.grad)


@pytest.mark.parametrize("eight", [False, True])
def test_training_then_decoding_sees_the_new_weights_and_statistics(vae, eight):
    """The decoder kernel's packed weights follow a training step on the layer operators, running statistics
    included, which those write behind torch's back."""
    _, b = pair(vae, dropout=0.15, checkpoint8=eight)
    x, c, z = batch(256)
    b.eval()
    with torch.no_grad():
        before = b.decode(z, c)
    b.train()
    opt = torch.optim.SGD(b.parameters(), lr=1e-2)
    mean, std = torch.zeros(5, device="cuda"), torch.ones(5, device="cuda")
    recon, mu, logvar = b(x, c)
    loss = b.loss_function(recon, x, mu, logvar, mean, std)[0]
    loss.backward()
    opt.step()
    b.eval()
    with torch.no_grad():
        after, ref = b.decode(z, c), b.decoder(torch.cat([z, c], dim=1))
        assert not torch.equal(before, after)
        near(after, ref, "decode after a step")
        b.train()
        b._run_stack(b.decoder, torch.cat([z, c], dim=1))        # statistics alone move
        b.eval()
        near(b.decode(z, c), b.decoder(torch.cat([z, c], dim=1)), "decode after new statistics")


def test_refusals(vae):
    with pytest.raises(ValueError):
        vae(checkpoint8=True)
    m = vae(layer_kernels=True).train()
    x, c, z = (t.cpu() for t in batch(4))
    for call in (lambda: m.encode(x, c), lambda: m.decode(z, c)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    m = m.cuda()
    with pytest.raises(ValueError, match="more than one row"):
        m.encode(x[:1].cuda(), c[:1].cuda())
