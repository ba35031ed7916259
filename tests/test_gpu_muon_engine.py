"""The optimizer step with orthogonalised momentum inside VoxelEngine, and the new operators run together as a training step uses them: head
norm + rotation between the qkv product and the attention, its backward, and the update of the qkv weight."""
import pytest
import torch

from simple3d_former_amd import _lib as L
from simple3d_former_amd import ops
from tests.test_gpu_muon import check_muon

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import simple3d_former_amd as s3d
    from oracle import voxel_oracle as vo

DEV = 'cuda'
KW = dict(backbone='deit_tiny_patch16_224', embed_layer='VoxelEmbed', voxel_size=12, cell=4, patch=3, n_classes=10)
GROUP = dict(KW, embed_layer='VoxelEmbed_no_average', pos_embedding='group_embed')


def engines(n, kw=KW, **more):
    sd = vo.init_state_dict(seed=1, exercise_all=True, **kw)
    x, y = vo.synthetic_batch(4, 12, 10, seed=2)
    out = []
    for _ in range(n):
        e = s3d.VoxelEngine(device='cuda:0', **kw, **more)
        e.load_state_dict(sd)
        out.append(e)
    return out, x.to(DEV), y.to(DEV)


@pytest.mark.parametrize('kw', [KW, GROUP])
def test_matrices_take_the_orthogonalised_step_and_the_rest_adam(kw):
    (a, b), x, y = engines(2, kw)
    hyper = torch.tensor([2e-3, 0.9, 0.05, 0.5], device=DEV)
    a.set_muon(lr=2e-3, momentum=0.9, weight_decay=0.05, grad_scale=0.5)
    stacks = a.muon_stacks()
    assert sum(n for _, n, _, _, _ in stacks) == 4 * a.depth + (4 if a.group else 0)
    for e in (a, b):                                # the same gradients and moments in both (a backward with atomics need not repeat)
        e.forward(x)
        e.cross_entropy(4, y)
        e.zero_grad()
        e.backward(4)
    g = torch.Generator(device=DEV).manual_seed(0)
    b.arena.g.copy_(a.arena.g)
    m0 = torch.randn(a.arena.numel, generator=g, device=DEV) * 1e-3
    pad = torch.ones(a.arena.numel, dtype=torch.bool, device=DEV)
    for k in a.shapes:
        o = a.arena.offsets[k]
        pad[o:o + a.arena.param(k).numel()] = False
    m0[pad] = 0
    for e in (a, b):
        e.arena.m.copy_(m0)
    p0, g0 = a.arena.p.clone(), a.arena.g.clone()
    a.optimizer_step()
    b.adam_step()
    matrix = torch.zeros(a.arena.numel, dtype=torch.bool, device=DEV)
    for k, n, r, c, stride in stacks:
        for i in range(n):
            o = a.arena.offsets[k] + i * stride
            matrix[o:o + r * c] = True
            v = lambda t: t[o:o + r * c].view(r, c)
            check_muon(v(p0), v(g0), v(m0), v(a.arena.p), v(a.arena.m), hyper, True, ops.muon_scale('match_rms_adamw', r, c))
    rest = ~matrix
    for name in ('p', 'm', 'v', 'hi', 'lo'):
        assert torch.equal(getattr(a.arena, name)[rest], getattr(b.arena, name)[rest]), name      # bit for bit what Adam does
    assert bool((a.arena.v[matrix] == 0).all()) and bool((a.arena.g == 0).all()) and bool((a.arena.p[pad] == 0).all())
    assert torch.equal(a.arena.hi, a.arena.p.to(torch.bfloat16))
    assert torch.equal(a.arena.lo, (a.arena.p - a.arena.hi.float()).to(torch.bfloat16))
    assert a.optimizer_state()['step'] == 1


def test_train_step_eager_and_captured_and_back_to_adam():
    """A captured step follows the learning rate on the device; eager and replayed steps agree to the backward's own repeatability
    (deterministic mode: bit for bit); set_muon / unset_muon choose the capture."""
    L.lib().s3d_set_deterministic(1)
    try:
        (a, b), x, y = engines(2)
        for e in (a, b):
            e.set_muon(lr=1e-3, momentum=0.95)
        graph, sx, sy, loss = b.capture_train_step(4)
        sx.copy_(x)
        sy.copy_(y)
        for k in range(3):
            for e in (a, b):
                e.set_muon(lr=1e-3 / (k + 1))
            la = a.train_step(x, y)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(a.arena.p, b.arena.p) and torch.equal(a.arena.m, b.arena.m) and float(la) == float(loss), k
        assert b.capture_train_step(4)[0] is graph
        p = a.arena.p.clone()
        for e in (a, b):
            e.unset_muon()
        adam_graph = b.capture_train_step(4)
        assert adam_graph[0] is not graph
        adam_graph[1].copy_(x)
        adam_graph[2].copy_(y)
        a.train_step(x, y)
        adam_graph[0].replay()
        torch.cuda.synchronize()
        assert torch.equal(a.arena.p, b.arena.p) and not torch.equal(a.arena.p, p)
    finally:
        L.lib().s3d_set_deterministic(0)


def test_refusals():
    (a,), x, y = engines(1)
    with pytest.raises(RuntimeError, match='set_muon first'):
        a.muon_step()
    a.set_muon()
    for call in (a.adam_step, lambda: a.adam_apply(0, 512)):
        with pytest.raises(RuntimeError, match='set_muon is in effect'):
            call()
    with pytest.raises(ValueError):
        a.set_muon(scale='unknown rule')
    a.unset_muon()
    a.adam_step()
    with pytest.raises(ValueError, match='current device'):
        ops.muon_step([torch.zeros(3, 4)], [torch.zeros(3, 4)], [torch.zeros(3, 4)], torch.zeros(4))
    d = lambda *s: torch.zeros(*s, device=DEV)
    with pytest.raises(ValueError, match='differ'):
        ops.muon_step([d(3, 4)], [d(4, 3)], [d(3, 4)], d(4))
    with pytest.raises(ValueError, match='4 values'):
        ops.muon_step([d(3, 4)], [d(3, 4)], [d(3, 4)], d(3))
    with pytest.raises(ValueError, match='laid out like'):
        ops.muon_step([d(3, 4)], [d(3, 4)], [d(3, 4)], d(4), planes=[(d(3, 5).bfloat16()[:, :4], d(3, 4).bfloat16())])
    with pytest.raises(ValueError, match='contiguous'):
        ops.orthogonalize(d(4, 6).t())
    with pytest.raises(ValueError, match='float32 / torch.bfloat16'):
        ops.orthogonalize(d(4, 6).half())
    with pytest.raises(RuntimeError, match='overlap'):
        ops.orthogonalize(d(2, 4, 6), out=d(1, 4, 6).expand(2, 4, 6))
    h = torch.zeros(4, 576, device=DEV, dtype=torch.bfloat16)
    for bad in (dict(rope=(d(4, 32), d(4, 31))), dict(rope=(d(4, 32).double(), d(4, 32))), dict(pos=torch.zeros(3, dtype=torch.int32, device=DEV)),
                dict(pos=torch.zeros(4, dtype=torch.int64, device=DEV)), dict(q_gain=d(63)), dict(out=(h[:3], None)), dict(Hkv=2)):
        with pytest.raises(ValueError):
            ops.qk_norm_rope_fwd(h, None, 3, 64, **bad)
    with pytest.raises(RuntimeError, match='aligned'):
        ops.qk_norm_rope_fwd(torch.zeros(4 * 584, device=DEV, dtype=torch.bfloat16)[4:4 + 4 * 576].view(4, 576), None, 3, 64)


def test_head_norm_attention_and_update_run_together():
    """x -> qkv -> head norm + rotation by grid coordinates -> attention -> loss, back through all of it, then one optimizer step on the qkv
    weight: gradients against 64-bit autograd, the update against the rule on the device's own gradient."""
    B, N, H, hd = 5, 28, 3, 64
    D, rows = H * hd, B * N
    g = torch.Generator().manual_seed(0)
    x = torch.randn(rows, D, generator=g).to(DEV)
    W = (torch.randn(3 * D, D, generator=g) * D ** -0.5).to(DEV)
    wout = torch.randn(rows, D, generator=g).to(DEV).to(torch.bfloat16)
    gq, gk = [(1.5 + 0.2 * torch.randn(hd, generator=g)).to(DEV) for _ in range(2)]
    # 27 cells of a 3 x 3 x 3 grid behind a class token without a position
    cells = torch.stack(torch.meshgrid(*[torch.arange(3)] * 3, indexing='ij'), -1).reshape(-1, 3)
    rope = tuple(t.to(DEV) for t in ops.rope_table(cells, hd))
    pos = torch.cat([torch.tensor([-1]), torch.arange(27)]).repeat(B).to(torch.int32).to(DEV)

    def step():
        qkv = ops.split_bf16(ops.linear(x, W, None, split=True))
        nrm = ops.qk_norm_rope_fwd(qkv[0], qkv[1], H, hd, q_gain=gq, k_gain=gk, rope=rope, pos=pos)
        out_hi, out_lo, lse = ops.attention_fwd(nrm[0], nrm[1], B, H, N, D, N, 1)
        dnrm = ops.attention_bwd(nrm[0], out_hi, out_lo, lse, wout, B, H, N, D, N, 1)
        dqkv, _, dgq, dgk = ops.qk_norm_rope_bwd(dnrm, None, qkv[0], qkv[1], H, hd, q_gain=gq, k_gain=gk, rope=rope, pos=pos)
        dW = torch.zeros(3 * D, D, device=DEV)
        ops.gemm(1, 1, False, 'ATOMIC', A_hi=dqkv, lda=3 * D, B_hi=ops.split_bf16(x)[0], ldb=D, M=3 * D, N=D, K=rows, C=dW, ldc=D)
        return out_hi.double() + out_lo.double(), dW, dgq, dgk
    out, dW, dgq, dgk = step()
    # the same in 64 bits
    Wr, gqr, gkr = (t.double().requires_grad_() for t in (W, gq, gk))
    q, k, v = (x.double() @ Wr.T).view(B, N, 3, H, hd).permute(2, 0, 3, 1, 4)
    on = (pos >= 0).view(B, 1, N, 1)
    cos, sin = (torch.where(on, t.double()[pos.long().clamp(min=0)].view(B, 1, N, hd // 2), e) for t, e in zip(rope, (1.0, 0.0)))

    def norm(t, gain):
        z = t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * gain
        a, b = z.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    s = torch.softmax(torch.matmul(norm(q, gqr), norm(k, gkr).transpose(-1, -2).contiguous()) * hd ** -0.5, -1)
    ref = torch.matmul(s, v).permute(0, 2, 1, 3).reshape(rows, D)
    rW, rq, rk = torch.autograd.grad((ref * wout.double()).sum(), [Wr, gqr, gkr])
    # forward: split operands (2^-16) through a softmax over logits of a few units; backward: plain bf16 operands, a handful of roundings of 2^-9 rms
    assert float((out - ref.detach()).norm() / ref.detach().norm()) < 1e-4
    for got, want in ((dW, rW), (dgq, rq), (dgk, rk)):
        assert float((got.double() - want).norm() / want.norm()) < 2e-2
    m = torch.zeros_like(W)
    hyper = torch.tensor([1e-2, 0.95, 0.1, 1.0], device=DEV)
    W0 = W.clone()
    # the three projections of the packed weight are three matrices of one stack
    three = lambda t: t.view(3, D, D)
    ops.muon_step([three(W)], [three(dW)], [three(m)], hyper)
    check_muon(three(W0), three(dW), torch.zeros(3, D, D, device=DEV), three(W), three(m), hyper, True, 1.0)
