"""Overlapping tensors that the head norm and the orthogonalised updates refuse (checked before anything is launched: no GPU, no pointer followed)."""
import pytest

from simple3d_former_amd import _lib as L
from tests.test_operators_refusals import A, P, items, lib, ns, ortho, refused      # noqa: F401  (lib: the fixture)


@pytest.mark.parametrize('second', [
    dict(x=2 * A + 800, x_stride=-200, out=5 * A),                                # backwards over the first item's output
    dict(x=2 * A + 2400, x_stride=-400, out=5 * A),                               # ... its first matrix alone
    dict(x=2 * A + 400, x_stride=-(1 << 10), out=5 * A),
    dict(x=2 * A + 40, x_stride=-1, out=5 * A, count=1)])                        # one matrix: its stride says nothing
def test_inputs_that_run_backwards_through_another_output_are_refused(lib, second):      # noqa: F811
    f = [dict(dict(x=A, out=2 * A), **kw) for kw in ({}, second)]
    refused(lib.s3d_orthogonalize(items(L.S3dOrthoItem, ortho, *f), 2, ns(), P, 1 << 40, None), lib, 'shares memory')
