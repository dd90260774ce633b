"""CPU tests of how the drop-in conditional VAE strings the layer operators together (layer_kernels=True): the modules'
own modes, against the torch stack itself.  The operators are replaced by their formulas in torch; the kernels behind them
have tests of their own."""
import importlib
import sys

import pytest
import torch
import torch.nn.functional as F

import afiv_bootstrap


@pytest.fixture()
def cvae(monkeypatch):
    for p in afiv_bootstrap.dropin_paths():
        if p not in sys.path:
            sys.path.insert(0, p)
    module = importlib.import_module("cvae_model")
    acts = {"none": lambda z: z, "relu": torch.relu, "leaky_relu": lambda z: F.leaky_relu(z, 0.2), "tanh": torch.tanh}

    def linear_act(x, weight, bias=None, residual=None, act="none", checkpoint8=False):
        return acts[act](F.linear(x, weight, bias))

    def batch_norm_act(x, weight, bias, running_mean=None, running_var=None, act="none", keep=None, drop_p=0.0, momentum=0.1, eps=1e-5, checkpoint8=False):
        assert (keep is None) == (drop_p == 0.0) and 0.0 <= drop_p < 1.0 and isinstance(momentum, float)
        y = acts[act](F.batch_norm(x, running_mean, running_var, weight, bias, True, momentum, eps))
        return y if keep is None else y * keep / (1 - drop_p)
    monkeypatch.setattr(module._afiv, "linear_act", linear_act)
    monkeypatch.setattr(module._afiv, "batch_norm_act", batch_norm_act)
    return module


def pair(cvae, **kw):
    torch.manual_seed(3)
    a = cvae.ConditionalVAE_SingleHeston(**kw).double()
    b = cvae.ConditionalVAE_SingleHeston(layer_kernels=True, **kw).double()
    for m in a.modules():
        if isinstance(m, torch.nn.BatchNorm1d):
            m.running_mean.normal_(), m.running_var.uniform_(0.5, 2.0)
    b.load_state_dict(a.state_dict())
    return a, b


def modes(model, norm, dropout):
    """Each kind of layer in its own mode."""
    model.train()
    for m in model.modules():
        if isinstance(m, torch.nn.BatchNorm1d):
            m.train(norm)
        if isinstance(m, torch.nn.Dropout):
            m.train(dropout)


def close(a, b, what=""):
    # the same few sums of 64-bit numbers in another order
    assert torch.allclose(a, b, rtol=1e-9, atol=1e-11), (what, float((a - b).abs().max()))


@pytest.mark.parametrize("p", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("norm,dropout", [(True, False), (False, True), (False, False), (True, True)])
def test_each_layer_follows_its_own_mode(cvae, norm, dropout, p):
    a, b = pair(cvae, dropout=p)
    h = torch.randn(40, 13, dtype=torch.float64)
    outs = []
    for model, run in ((a, lambda m: m.encoder(h)), (b, lambda m: m._run_stack(m.encoder, h))):
        modes(model, norm, dropout)
        torch.manual_seed(8)
        outs.append(run(model))
        again = run(model)
        assert torch.equal(outs[-1], again) == (not dropout or p in (0.0, 1.0))      # a mask is drawn anew, or there is none
    if norm and dropout and 0.0 < p < 1.0:                   # other masks from the same generator: as many zeros, about
        zeros = [float((o == 0).double().mean()) for o in outs]
        assert abs(zeros[0] - zeros[1]) < 0.12, zeros        # six standard deviations of the difference over 1280 elements
    else:
        close(*outs)
    for (name, u), v in zip(b.named_buffers(), a.buffers()):
        if not (norm and dropout and 0.0 < p < 1.0):
            close(u.double(), v.double(), name)


def test_gradients_with_frozen_statistics_and_dropout(cvae):
    a, b = pair(cvae, dropout=0.5)
    h = torch.randn(40, 13, dtype=torch.float64)
    for model, run in ((a, lambda m: m.encoder(h)), (b, lambda m: m._run_stack(m.encoder, h))):
        modes(model, False, True)
        torch.manual_seed(8)
        run(model).square().sum().backward()
    for (name, u), v in zip(b.encoder.named_parameters(), a.encoder.parameters()):
        close(u.grad, v.grad, name)


@pytest.mark.parametrize("momentum,tracks", [(None, True), (0.3, True), (0.1, False), (None, False)])
def test_running_statistics_rules_of_the_module(cvae, momentum, tracks):
    a, b = pair(cvae, dropout=0.0)
    for model in (a, b):
        for m in model.modules():
            if isinstance(m, torch.nn.BatchNorm1d):
                m.momentum, m.track_running_stats = momentum, tracks
    batches = [torch.randn(20, 13, dtype=torch.float64) + i for i in range(3)]
    for model, run in ((a, lambda h: a.encoder(h)), (b, lambda h: b._run_stack(b.encoder, h))):
        model.train()
        for h in batches:
            run(h)
    for (name, u), v in zip(b.named_buffers(), a.buffers()):
        close(u.double(), v.double(), name)
    a.eval(), b.eval()
    close(b._run_stack(b.encoder, batches[0]), a.encoder(batches[0]))


def test_statistics_that_are_not_kept(cvae):
    """Without running statistics the batch's own serve in evaluation too."""
    a, b = pair(cvae, dropout=0.0)
    for model in (a, b):
        for m in model.modules():
            if isinstance(m, torch.nn.BatchNorm1d):
                m.track_running_stats, m.running_mean, m.running_var, m.num_batches_tracked = False, None, None, None
    h = torch.randn(20, 13, dtype=torch.float64)
    for mode in (True, False):
        a.train(mode), b.train(mode)
        close(b._run_stack(b.encoder, h), a.encoder(h))


@pytest.mark.parametrize("register", ["register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook", "register_full_backward_pre_hook"])
def test_hooks_are_refused_not_skipped(cvae, register):
    """The modules are never called, so a hook on one of them could not run."""
    _, b = pair(cvae, dropout=0.5)
    h = torch.randn(20, 13, dtype=torch.float64)
    for module, call in [(m, lambda: b._run_stack(b.encoder, h)) for m in (b.encoder, *b.encoder)] + [(b.fc_mu, lambda: b._linear(b.fc_mu, h[:, :b.fc_mu.in_features]))]:
        handle = getattr(module, register)(lambda *args: None)
        with pytest.raises(RuntimeError, match="hooks"):
            call()
        handle.remove()
    assert b._run_stack(b.encoder, h).shape[0] == 20


def test_another_slope_is_refused(cvae):
    """The operators' leaky_relu has one slope; the module's may be set."""
    _, b = pair(cvae, dropout=0.0, encoder_activation="leaky_relu")
    h = torch.randn(20, 13, dtype=torch.float64)
    b._run_stack(b.encoder, h)
    next(m for m in b.encoder if isinstance(m, torch.nn.LeakyReLU)).negative_slope = 0.1
    with pytest.raises(ValueError, match="slope"):
        b._run_stack(b.encoder, h)


def test_models_pickled_without_the_option(cvae):
    """A whole model pickled before the option existed has none of its attributes: it runs on its torch layers."""
    a, _ = pair(cvae, dropout=0.0)
    del a.__dict__["layer_kernels"], a.__dict__["checkpoint8"]
    a.train()
    x, c, z = (torch.randn(6, k, dtype=torch.float64) for k in (5, 8, 4))
    a.encode(x, c)
    a.decode(z, c)
