"""Gains and their gradients that lie between the rows of a pitched output share no element with it: such calls are taken."""
import pytest
import torch

from simple3d_former_amd import ops
from tests.test_gpu_qk_norm import DEV, gains, make, table

pytestmark = pytest.mark.gpu


def test_gains_and_gradients_between_the_rows_of_the_output():
    rows, H, hd = 6, 3, 64
    W = 3 * H * hd
    hi, _ = make(rows, H, H, hd, False)
    d, _ = make(rows, H, H, hd, False, seed=1)
    gq, gk = gains(hd)
    rope = table(rows, hd)
    kw = dict(q_gain=gq, k_gain=gk, rope=rope)
    want = ops.qk_norm_rope_fwd(hi, None, H, hd, **kw)[0]
    grads = ops.qk_norm_rope_bwd(d, None, hi, None, H, hd, **kw)
    buf = torch.zeros(rows, W + 512, dtype=torch.bfloat16, device=DEV)             # 1024 bytes behind every row: room for four vectors
    gap = buf.view(torch.float32)[2, W // 2:].view(4, hd)
    gap[0], gap[1] = gq, gk
    out = buf[:, :W]
    got = ops.qk_norm_rope_fwd(hi, None, H, hd, q_gain=gap[0], k_gain=gap[1], rope=rope, out=(out, None))[0]
    assert torch.equal(got, want)
    got = ops.qk_norm_rope_bwd(d, None, hi, None, H, hd, q_gain=gap[0], k_gain=gap[1], rope=rope, out=(out, None), gain_grads=(gap[2], gap[3]))
    assert torch.equal(got[0], grads[0]) and torch.equal(gap[2], grads[2]) and torch.equal(gap[3], grads[3])
    assert torch.equal(gap[0], gq) and torch.equal(gap[1], gk)
    with pytest.raises(RuntimeError, match='overlap'):                             # the last 256 bytes of a row
        ops.qk_norm_rope_fwd(hi, None, H, hd, q_gain=buf.view(torch.float32)[2, W // 2 - hd:W // 2], rope=rope, out=(out, None))
    with pytest.raises(RuntimeError, match='overlap'):                             # gradients added to the gains themselves
        ops.qk_norm_rope_bwd(d, None, hi, None, H, hd, q_gain=gq, k_gain=gk, gain_grads=(gq, gk))
