"""The data-parallel trainers update slices of the arena with Adam: with set_muon in effect they refuse before a step begins, not behind its backward and
its collectives."""
from types import SimpleNamespace

import pytest
import torch

from simple3d_former_amd.parallel import DataParallelTrainer, ShardedDataParallelTrainer


class Untouched:
    """An engine with set_muon in effect; anything but that setting is out of bounds."""
    muon = (True, 5, (3.4445, -4.7750, 2.0315), 'original')

    def __getattr__(self, name):
        raise AssertionError(f'the step went on to engine.{name}')


@pytest.mark.parametrize('cls', [DataParallelTrainer, ShardedDataParallelTrainer])
@pytest.mark.parametrize('call', ['step_eager', 'step', 'graph step', 'capture'])
def test_refused_before_anything_runs(cls, call):
    t = object.__new__(cls)                                  # (a constructor needs an engine on a GPU)
    t.eng, t._cap, t.use_graphs, t.pending, t.slices, t.segments = Untouched(), None, call == 'graph step', False, [(0, 8)], [(0, 0)]
    t.fwd_ranges, t.shards, t.world, t.graph_collectives, t.sliced_adam = [(0, 0)], [(0, 8)], 1, False, True
    t.reducer = SimpleNamespace(force=False)
    x, y = torch.zeros(2, 1, 4, 4, 4), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match='set_muon is in effect'):
        t.capture(2) if call == 'capture' else t.step_eager(x, y) if call == 'step_eager' else t.step(x, y)
