"""What the head norm and the orthogonalised updates refuse: arguments are checked before anything is launched, so this runs without a GPU
(the pointers below are never followed)."""
import ctypes
import os

import pytest
import torch

from simple3d_former_amd import _lib as L
from simple3d_former_amd import ops

P = 0x1000          # 16-byte aligned, never dereferenced


@pytest.fixture(scope='module')
def lib():
    if not os.path.exists(L.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    return L.lib()


def refused(rc, lib, text):
    assert rc != 0
    assert text in lib.s3d_last_error_string().decode(), lib.s3d_last_error_string()


def qk(**kw):
    f = dict(qkv_hi=P, ld=576, out_hi=2 * P, ldo=576, rows=10, H=3, Hkv=3, hd=64, eps=1e-6, st=1)
    f.update(kw)
    return ctypes.byref(L.fill(L.S3dQkNormArgs(), **f))


@pytest.mark.parametrize('kw,text', [
    (dict(hd=60), 'head dim'), (dict(hd=8), 'head dim'), (dict(hd=272), 'head dim'), (dict(H=0), 'heads'), (dict(Hkv=0), 'heads'), (dict(rows=-1), 'rows'),
    (dict(rows=1 << 31), 'rows'), (dict(ld=570), 'pitch'), (dict(ld=580), 'pitch'), (dict(ldo=512), 'pitch'), (dict(qkv_hi=0), 'aligned'), (dict(qkv_hi=P + 2), 'aligned'),
    (dict(out_hi=0), 'aligned'), (dict(out_hi=P + 8), 'aligned'), (dict(qkv_lo=P + 4), 'aligned'), (dict(eps=-1.0), 'eps'), (dict(eps=float('nan')), 'eps'),
    (dict(cos_t=P), 'both tables'), (dict(cos_t=P, sin_t=P, T=0), 'tables'), (dict(cos_t=P, sin_t=P + 4, T=5), 'tables'), (dict(cos_t=P, sin_t=P, T=5, st=0), 'stride'),
    (dict(out_hi=P, ldo=640), 'in place'), (dict(out_hi=P, out_lo=3 * P), 'in place')])
def test_qk_norm_forward_refuses(lib, kw, text):
    refused(lib.s3d_qk_norm_rope_fwd(qk(**kw), None), lib, text)


@pytest.mark.parametrize('kw,text', [
    (dict(dout=0), 'dout'), (dict(dqkv=0), 'dqkv'), (dict(lddo=500), 'pitch'), (dict(lddq=577), 'pitch'), (dict(dq_gain=0), 'dq_gain'), (dict(partial=0), 'partial'),
    (dict(partial_blocks=0), 'partial'), (dict(dqkv=3 * P, lddq=640), 'in place'), (dict(dout_lo=P + 2), 'aligned'), (dict(hd=24), 'head dim')])
def test_qk_norm_backward_refuses(lib, kw, text):
    f = dict(dout=3 * P, lddo=576, dqkv=4 * P, lddq=576, dq_gain=P, dk_gain=P, partial=P, partial_blocks=1)
    f.update(kw)
    refused(lib.s3d_qk_norm_rope_bwd(qk(**f), None), lib, text)


def test_null_args_and_sizes(lib):
    for fn in (lib.s3d_qk_norm_rope_fwd, lib.s3d_qk_norm_rope_bwd):
        refused(fn(None, None), lib, 'null args')
    refused(lib.s3d_orthogonalize(None, 1, None, None, 0, None), lib, 'null args')
    refused(lib.s3d_muon_step(None, 1, None, None, None, 0, None), lib, 'null args')
    assert lib.s3d_qk_norm_rope_fwd(qk(rows=0), None) == 0                     # no rows: nothing is launched
    assert lib.s3d_qk_norm_blocks(0, 3, 3, 64) == 0 and lib.s3d_qk_norm_blocks(1, 3, 3, 64) == 1
    assert lib.s3d_orthogonalize_workspace_bytes(None, 1, None) == 0


def ns(**kw):
    f = dict(steps=5, a=3.4445, b=-4.7750, c=2.0315, eps=1e-7)
    f.update(kw)
    return ctypes.byref(L.fill(L.S3dNsArgs(), **f))


def ortho(**kw):
    f = dict(x=P, x_stride=0, x_ld=20, out=2 * P, out_stride=200, out_ld=20, count=2, rows=10, cols=20)
    f.update(kw)
    return (L.S3dOrthoItem * 1)(L.fill(L.S3dOrthoItem(), **f))


def muon(**kw):
    f = dict(p=P, p_stride=200, p_ld=20, g=2 * P, g_stride=200, g_ld=20, m=3 * P, m_stride=200, m_ld=20, count=2, rows=10, cols=20, scale=1.0)
    f.update(kw)
    return (L.S3dMuonItem * 1)(L.fill(L.S3dMuonItem(), **f))


@pytest.mark.parametrize('kw,text', [
    (dict(steps=0), 'steps'), (dict(steps=33), 'steps'), (dict(a=float('nan')), 'coefficients'), (dict(b=float('inf')), 'coefficients'), (dict(eps=0.0), 'eps'),
    (dict(eps=float('nan')), 'eps'), (dict(a=100.0), 'polynomial'), (dict(a=4.0, b=0.0, c=0.0), 'polynomial')])
def test_newton_schulz_refuses(lib, kw, text):
    it = ortho()
    refused(lib.s3d_orthogonalize(it, 1, ns(**kw), P, 1 << 30, None), lib, text)
    refused(lib.s3d_muon_step(muon(), 1, ns(**kw), P, P, 1 << 30, None), lib, text)


@pytest.mark.parametrize('kw,text', [
    (dict(x=0), 'null pointer'), (dict(out=0), 'null pointer'), (dict(rows=-1), 'negative'), (dict(cols=1 << 17, x_ld=1 << 17, out_ld=1 << 17), 'too large'),
    (dict(x_ld=19), 'pitch'), (dict(out_ld=19), 'pitch'), (dict(out_stride=199), 'overlap'), (dict(out_stride=0), 'overlap')])
def test_orthogonalize_refuses_items(lib, kw, text):
    refused(lib.s3d_orthogonalize(ortho(**kw), 1, ns(), P, 1 << 40, None), lib, text)


@pytest.mark.parametrize('kw,text', [
    (dict(p=0), 'null pointer'), (dict(g=0), 'null pointer'), (dict(m=0), 'null pointer'), (dict(hi=P), 'planes'), (dict(lo=P), 'planes'), (dict(p_ld=10), 'pitch'),
    (dict(g_ld=10), 'pitch'), (dict(m_ld=10), 'pitch'), (dict(p_stride=100), 'overlap'), (dict(m_stride=0), 'overlap'), (dict(g_stride=0), 'overlap'),
    (dict(scale=float('inf')), 'scale')])
def test_muon_refuses_items(lib, kw, text):
    refused(lib.s3d_muon_step(muon(**kw), 1, ns(), P, P, 1 << 40, None), lib, text)


def test_workspace_is_checked(lib):
    need = lib.s3d_orthogonalize_workspace_bytes(ortho(), 1, ns())
    assert need > 0
    refused(lib.s3d_orthogonalize(ortho(), 1, ns(), P, need - 1, None), lib, 'workspace')
    refused(lib.s3d_orthogonalize(ortho(), 1, ns(), None, need, None), lib, 'workspace')
    refused(lib.s3d_orthogonalize(ortho(), 1, ns(), P + 4, need, None), lib, 'workspace')
    need = lib.s3d_muon_workspace_bytes(muon(), 1, ns())
    refused(lib.s3d_muon_step(muon(), 1, ns(), P, P, need - 1, None), lib, 'workspace')
    refused(lib.s3d_muon_step(muon(), 1, ns(), None, P, need, None), lib, 'hyper')
    # items without elements need no pointers and launch nothing
    assert lib.s3d_orthogonalize(ortho(x=0, out=0, count=0), 1, ns(), P, 256, None) == 0


def test_wrappers_refuse():
    x = torch.zeros(4, 576, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match='current device'):
        ops.qk_norm_rope_fwd(x, None, 3, 64)
    with pytest.raises(ValueError, match='current device'):
        ops.orthogonalize(torch.zeros(4, 5))
    with pytest.raises(ValueError, match='same length'):
        ops.muon_step([torch.zeros(2, 2)], [], [], torch.zeros(4))
    with pytest.raises(ValueError, match='head dim'):
        ops.rope_table(torch.arange(4), 40)
    with pytest.raises(ValueError, match='axes'):
        ops.rope_table(torch.zeros(4, 9), 16)
    assert ops.muon_scale('original', 8, 2) == 2.0 and ops.muon_scale('original', 2, 8) == 1.0
    assert ops.muon_scale('match_rms_adamw', 25, 100) == 2.0 and ops.muon_scale(0.5, 3, 3) == 0.5


@pytest.mark.parametrize('kw', [
    dict(out_hi=P + 16), dict(out_hi=P + 576 * 8), dict(qkv_lo=1 << 20, out_hi=1 << 20, out_lo=P), dict(out_lo=2 * P), dict(out_lo=2 * P + 64)])
def test_qk_norm_forward_refuses_overlapping_planes(lib, kw):
    """Rows of 576 elements, ten of them: 11520 bytes.  Shifted planes, swapped planes, one plane for both halves of a pair."""
    f = dict(out_hi=1 << 22)
    f.update(kw)
    refused(lib.s3d_qk_norm_rope_fwd(qk(**f), None), lib, 'overlap')


@pytest.mark.parametrize('kw', [
    dict(dk_gain=1 << 23), dict(dk_gain=(1 << 23) + 128), dict(dqkv=(1 << 22) + 1152), dict(dqkv=P + 16), dict(dqkv_lo=(1 << 22) + (1 << 14))])
def test_qk_norm_backward_refuses_overlapping_tensors(lib, kw):
    """One gradient tensor for both gains (two workgroups would add to it), shifted planes."""
    f = dict(out_hi=0, dout=1 << 21, lddo=576, dqkv=(1 << 22) + (1 << 14), lddq=576, dq_gain=1 << 23, dk_gain=1 << 24, partial=P, partial_blocks=1)
    if 'dqkv' in kw and kw['dqkv'] != P + 16:
        f['dout'] = 1 << 22
    f.update(kw)
    refused(lib.s3d_qk_norm_rope_bwd(qk(**f), None), lib, 'overlap')


def items(cls, make, *kws):
    arr = (cls * len(kws))()
    for i, kw in enumerate(kws):
        arr[i] = make(**kw)[0]
    return arr


A = 1 << 20          # one tensor of 2 matrices [10][20]: 1600 bytes


@pytest.mark.parametrize('first,second', [
    (dict(), dict()),                                                           # the same parameter twice
    (dict(), dict(p=4 * A, g=5 * A)),                                           # one momentum for two parameters
    (dict(), dict(p=A + 800, g=5 * A, m=6 * A, count=1)),                       # a stack and its second matrix
    (dict(), dict(p=A + 40, g=5 * A, m=6 * A, count=1)),                        # columns that wrap into the next row
    (dict(), dict(p=4 * A, g=5 * A, m=A)),                                      # one's momentum, the other's parameter
    (dict(), dict(p=4 * A, g=A, m=6 * A)),                                      # one's parameter, the other's gradient
    (dict(g=A), dict(p=4 * A, g=5 * A, m=6 * A)),                               # parameter and gradient of one item
    (dict(hi=8 * A, lo=8 * A), dict(p=4 * A, g=5 * A, m=6 * A)),                # one plane for both halves
    (dict(hi=8 * A, lo=A), dict(p=4 * A, g=5 * A, m=6 * A))])                   # a plane in the parameter
def test_muon_refuses_shared_tensors(lib, first, second):
    f = [dict(dict(p=A, g=2 * A, m=3 * A), **kw) for kw in (first, second)]
    refused(lib.s3d_muon_step(items(L.S3dMuonItem, muon, *f), 2, ns(), P, P, 1 << 40, None), lib, 'shares memory')


def test_muon_refuses_one_gradient_for_two_parameters_when_it_is_cleared(lib):
    f = [dict(p=A, g=2 * A, m=3 * A), dict(p=4 * A, g=2 * A, m=6 * A)]
    refused(lib.s3d_muon_step(items(L.S3dMuonItem, muon, *f), 2, ns(zero_grad=1), P, P, 1 << 40, None), lib, 'shares memory')


@pytest.mark.parametrize('second', [dict(x=4 * A), dict(x=4 * A, out=2 * A + 80), dict(x=2 * A + 400, out=5 * A, count=1)])
def test_orthogonalize_refuses_shared_outputs(lib, second):
    f = [dict(dict(x=A, out=2 * A), **kw) for kw in ({}, second)]
    refused(lib.s3d_orthogonalize(items(L.S3dOrthoItem, ortho, *f), 2, ns(), P, 1 << 40, None), lib, 'shares memory')


def test_no_items_are_no_work(lib):
    """An empty list needs no workspace: what the size calls say (0) is enough."""
    assert lib.s3d_muon_workspace_bytes(None, 0, ns()) == 0 and lib.s3d_orthogonalize_workspace_bytes(None, 0, ns()) == 0
    assert lib.s3d_muon_step(None, 0, ns(), P, None, 0, None) == 0
    assert lib.s3d_orthogonalize(None, 0, ns(), None, 0, None) == 0
    refused(lib.s3d_muon_step(None, 0, ns(steps=0), P, None, 0, None), lib, 'steps')
