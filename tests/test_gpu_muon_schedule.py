"""set_muon as a learning-rate schedule calls it: what is not given keeps its value, and a captured step stays the one in effect."""
import pytest
import torch

from simple3d_former_amd import ops
from tests.test_gpu_muon_engine import engines

pytestmark = pytest.mark.gpu


def test_a_schedule_keeps_the_other_settings():
    (e,), x, y = engines(1)
    e.set_muon(lr=1e-3, scale='original', steps=3, nesterov=False, coefficients=(1.875, -1.25, 0.375))
    muon, epoch = e.muon, e.capture_epoch
    graph = e.capture_train_step(4)[0]
    e.set_muon(lr=5e-4)
    assert e.muon == muon == (False, 3, (1.875, -1.25, 0.375), 'original') and e.capture_epoch == epoch and e.capture_train_step(4)[0] is graph
    assert float(e._muon_hyper[0]) == pytest.approx(5e-4)
    e.set_muon(steps=4)                                      # one of them changed
    assert e.muon == (False, 4, (1.875, -1.25, 0.375), 'original') and e.capture_epoch == epoch + 1
    e.unset_muon()
    e.set_muon()                                             # taken up anew: the defaults
    assert e.muon == (True, 5, ops.NS_COEFFICIENTS, 'match_rms_adamw')
