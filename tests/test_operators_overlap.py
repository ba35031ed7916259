"""Overlapping tensors that the head norm and the orthogonalised updates refuse (checked before anything is launched: no GPU, no pointer followed)."""
import pytest

from simple3d_former_amd import _lib as L
from tests.test_operators_refusals import A, P, items, lib, ns, ortho, qk, refused      # noqa: F401  (lib: the fixture)


@pytest.mark.parametrize('second', [
    dict(x=2 * A + 800, x_stride=-200, out=5 * A),                                # backwards over the first item's output
    dict(x=2 * A + 2400, x_stride=-400, out=5 * A),                               # ... its first matrix alone
    dict(x=2 * A + 400, x_stride=-(1 << 10), out=5 * A),
    dict(x=2 * A + 40, x_stride=-1, out=5 * A, count=1)])                        # one matrix: its stride says nothing
def test_inputs_that_run_backwards_through_another_output_are_refused(lib, second):      # noqa: F811
    f = [dict(dict(x=A, out=2 * A), **kw) for kw in ({}, second)]
    refused(lib.s3d_orthogonalize(items(L.S3dOrthoItem, ortho, *f), 2, ns(), P, 1 << 40, None), lib, 'shares memory')

FAR = 1 << 22          # rows of 576 elements, ten of them: 11520 bytes from here


@pytest.mark.parametrize('kw', [
    dict(q_gain=FAR), dict(k_gain=FAR + 11520 - 4), dict(q_gain=FAR - 252), dict(cos_t=FAR + 4096, sin_t=P, T=10), dict(cos_t=P, sin_t=FAR - 1264, T=10),
    dict(cos_t=P, sin_t=P, T=10, pos=FAR + 8), dict(cos_t=P, sin_t=P, T=10, pos=FAR - 36), dict(out_lo=2 * FAR, q_gain=2 * FAR + 1152),
    dict(ldo=640, q_gain=FAR + 1152 - 4), dict(ldo=640, q_gain=FAR + 1280 - 252)])
def test_forward_refuses_outputs_over_gains_tables_and_positions(lib, kw):      # noqa: F811
    f = dict(out_hi=FAR)
    f.update(kw)
    refused(lib.s3d_qk_norm_rope_fwd(qk(**f), None), lib, 'overlap')


def back(**kw):
    f = dict(out_hi=0, qkv_hi=1 << 20, dout=1 << 21, lddo=576, dqkv=FAR, lddq=576, dq_gain=1 << 23, dk_gain=1 << 24, partial=1 << 25, partial_blocks=10, q_gain=1 << 26,
             k_gain=1 << 27, cos_t=1 << 28, sin_t=1 << 29, T=10, pos=1 << 30)
    f.update(kw)
    return qk(**f)


@pytest.mark.parametrize('kw', [
    dict(q_gain=FAR), dict(pos=FAR + 11516), dict(cos_t=FAR - 1264),                                                # what is read, under dqkv
    dict(dq_gain=FAR), dict(dk_gain=FAR - 252), dict(partial=FAR + 11516), dict(partial=FAR - 508),                 # two things that are written
    dict(dq_gain=1 << 25), dict(dk_gain=(1 << 25) + 508),
    dict(dq_gain=1 << 20), dict(dk_gain=(1 << 21) + 11516), dict(partial=1 << 20), dict(partial=(1 << 21) + 11516),  # the planes that are read
    dict(dq_gain=1 << 26), dict(dk_gain=1 << 26), dict(dk_gain=1 << 28), dict(dq_gain=1 << 30), dict(partial=1 << 27), dict(partial=1 << 29), dict(partial=1 << 30)])
def test_backward_refuses_overlaps_of_everything_it_writes(lib, kw):      # noqa: F811
    refused(lib.s3d_qk_norm_rope_bwd(back(**kw), None), lib, 'overlap')
