"""VoxelEngine.set_muon refuses what the step would refuse, before anything is changed; a step that is refused all the same changes nothing."""
import pytest
import torch

from tests.test_gpu_muon_engine import engines

pytestmark = pytest.mark.gpu
NAN, INF = float('nan'), float('inf')
BAD = [dict(steps=0), dict(steps=33), dict(coefficients=(4.0, 0.0, 0.0)), dict(coefficients=(NAN, -4.775, 2.0315)), dict(coefficients=(3.0, INF, 2.0)),
       dict(coefficients=(1.5, -0.5)), dict(scale='unknown rule'), dict(scale=INF), dict(scale=NAN), dict(scale=1e39)]


def test_bad_settings_are_refused_and_change_nothing():
    (e,), x, y = engines(1)
    for kw in BAD:
        with pytest.raises((ValueError, RuntimeError)):
            e.set_muon(lr=0.5, **kw)
        assert e.muon is None, kw
    epoch = e.capture_epoch
    e.adam_step()                                            # Adam is still in effect
    e.set_muon(lr=2e-3, momentum=0.9)
    hyper, muon = e._muon_hyper.clone(), e.muon
    for kw in BAD:
        with pytest.raises((ValueError, RuntimeError)):
            e.set_muon(lr=0.5, momentum=0.1, **kw)
        assert e.muon == muon and torch.equal(e._muon_hyper, hyper) and e.capture_epoch == epoch + 1, kw
    e.train_step(x, y)
    assert e.optimizer_state()['step'] == 2


def test_a_refused_step_leaves_the_step_count_and_the_tensors():
    (e,), x, y = engines(1)
    e.set_muon()
    e.muon = (True, 0, e.muon[2], e.muon[3])                 # a setting that the step refuses
    e.arena.g.normal_(generator=torch.Generator(device='cuda').manual_seed(0))
    keep = [t.clone() for t in (e.arena.p, e.arena.g, e.arena.m, e.arena.v)]
    with pytest.raises(RuntimeError, match='steps'):
        e.muon_step()
    assert e.optimizer_state()['step'] == 0
    assert all(torch.equal(a, b) for a, b in zip(keep, (e.arena.p, e.arena.g, e.arena.m, e.arena.v)))
