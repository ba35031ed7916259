"""VoxelEngine between its two optimizers: what set_muon refuses, and what Adam finds when it takes the matrices back."""
import pytest
import torch

from tests.test_gpu_muon_engine import engines

pytestmark = pytest.mark.gpu


def adam_in_64_bits(p, g, m, v, t, lr, b1, b2, eps):
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + eps), m, v


@pytest.mark.parametrize('before', [0, 2])
def test_adam_begins_anew_behind_an_orthogonalised_step(before):
    """The second moments of the matrices are not kept up while set_muon is in effect, and the step count that Adam's bias corrections use is one for
    all parameters: behind unset_muon Adam starts from zero moments and step 1, an update of about lr an element instead of hundreds."""
    (e,), x, y = engines(1)
    lr, b1, b2, eps = 1e-3, 0.9, 0.999, 1e-8
    e.set_optimizer(lr=lr, betas=(b1, b2), eps=eps)
    for _ in range(before):                              # Adam, the orthogonalised step, Adam again
        e.train_step(x, y)
    e.set_muon(lr=1e-3, grad_scale=0.5)
    for _ in range(3):
        e.train_step(x, y)
    e.unset_muon()
    assert e.optimizer_state() == dict(lr=pytest.approx(lr), betas=pytest.approx((b1, b2)), eps=pytest.approx(eps), grad_scale=1.0, step=0)
    gen = torch.Generator(device='cuda').manual_seed(0)
    p = e.arena.p.double()
    m = v = torch.zeros_like(p)
    for t in (1, 2, 3):
        e.arena.g.zero_()
        for k in e.shapes:
            e.arena.grad(k).copy_(torch.randn(e.arena.grad(k).shape, generator=gen, device='cuda') * 1e-3)
        g, old = e.arena.g.double(), e.arena.p.double()
        e.optimizer_step()
        p, m, v = adam_in_64_bits(p, g, m, v, t, lr, b1, b2, eps)
        # 1 - 0.999 is formed in fp32: 2^-24 / 1e-3 of it, half under the root; everything else is a few roundings
        assert bool(((e.arena.p.double() - p).abs() <= t * (4 * 2.0 ** -24 * p.abs() + 1e-3 * lr)).all()), t
        assert float((e.arena.p.double() - old).abs().max()) <= 4 * lr, t


def test_moments_stay_where_no_orthogonalised_step_ran():
    (e,), x, y = engines(1)
    e.train_step(x, y)
    keep = e.arena.m.clone(), e.arena.v.clone()
    e.set_muon()
    e.unset_muon()
    assert torch.equal(e.arena.m, keep[0]) and torch.equal(e.arena.v, keep[1]) and e.optimizer_state()['step'] == 1


def test_replayed_steps_count_and_a_capture_alone_does_not():
    """A step of a cached capture runs no host code: Adam begins anew behind it all the same.  The capture itself restores what its warm-up changed."""
    (e,), x, y = engines(1)
    e.train_step(x, y)
    keep = e.arena.m.clone(), e.arena.v.clone()
    e.set_muon()
    graph, sx, sy, _ = e.capture_train_step(4)
    e.unset_muon()
    assert torch.equal(e.arena.m, keep[0]) and torch.equal(e.arena.v, keep[1]) and e.optimizer_state()['step'] == 1
    e.set_muon()
    e.set_muon(lr=2e-3)
    again = e.capture_train_step(4)
    assert again[0] is graph                                 # the capture of the first time
    sx.copy_(x), sy.copy_(y)
    graph.replay()
    e.set_optimizer(lr=1e-4, step=1)                         # (the count that set_muon found: a step ran all the same)
    e.unset_muon()
    assert not bool(e.arena.m.any()) and not bool(e.arena.v.any()) and e.optimizer_state()['step'] == 0
    assert e.optimizer_state()['lr'] == pytest.approx(1e-4)
