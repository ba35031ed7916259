"""Orthogonalised updates (s3d_orthogonalize, s3d_muon_step) against the same iteration in 64 bits, and against the singular values."""
import pytest
import torch

from simple3d_former_amd import ops

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
CO = ops.NS_COEFFICIENTS


def oracle(u, steps=5, co=CO, eps=1e-7):
    """[L, r, c] in 64 bits"""
    x = u.double()
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2) if tall else x
    x = x / torch.sqrt((x * x).sum((1, 2), keepdim=True)).clamp(min=eps)
    for _ in range(steps):
        a = torch.matmul(x, x.transpose(1, 2).contiguous())
        x = co[0] * x + torch.matmul(co[1] * a + co[2] * torch.matmul(a, a), x)
    return x.transpose(1, 2) if tall else x


def tol(steps):
    """Relative (2-norm) error.  A step rounds its operands three times to pairs of fp16 planes (2^-22 each) and drops lo x lo (2^-22); the map
    s -> a s + b s^3 + c s^5 multiplies an error that is there by at most its largest slope, 3.45 for small s."""
    return 4 * 2.0 ** -22 * sum(3.45 ** j for j in range(steps))


# Results in bf16: half a step (2^-8) of their own rounding, and the last two steps on single fp16 planes: X and P are rounded (2^-12 each) and the
# error multiplied by at most 3.45 a step up to the result.
BF16 = 2.0 ** -8 + 2 * 2.0 ** -12 * (3.45 ** 2 + 3.45)


def rel(got, want):
    got, want = got.double(), want.double()
    n = want.flatten(1).norm(dim=1)
    return float(((got - want).flatten(1).norm(dim=1) / n.clamp_min(1e-300)).max())


def grads(L, r, c, seed=0, dtype=torch.float32):
    """noise and a few strong directions: the spectrum of a gradient"""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(L, r, c, generator=g) + 0.25 * torch.randn(L, r, 8, generator=g) @ torch.randn(L, 8, c, generator=g)
    return (x * 1e-3).to(DEV, dtype)


SHAPES = [(1, 1, 1), (2, 1, 7), (2, 9, 1), (3, 5, 3), (1, 16, 16), (1, 64, 64), (2, 65, 64), (1, 63, 130), (2, 130, 63), (1, 192, 192), (2, 192, 576), (2, 576, 192),
          (1, 387, 1000), (1, 1000, 387), (3, 384, 384), (1, 768, 768), (1, 2, 5000), (1, 1031, 129), (5, 128, 256), (1, 129, 257), (2, 500, 100), (3, 90, 100),
          # enough tiles for the large ones: wide, tall, square, padded
          (12, 384, 1536), (12, 1536, 384), (2, 1536, 1530), (2, 1500, 1600), (9, 700, 640), (30, 250, 384), (130, 256, 520), (130, 520, 256)]


@pytest.mark.parametrize('L,r,c', SHAPES)
@pytest.mark.parametrize('src,dst', [('float32', 'float32'), ('bfloat16', 'bfloat16'), ('float32', 'bfloat16'), ('bfloat16', 'float32')])
def test_orthogonalize(L, r, c, src, dst):
    x = grads(L, r, c, dtype=getattr(torch, src))
    keep = x.clone()
    got = ops.orthogonalize(x, out_dtype=getattr(torch, dst))
    assert got.dtype == getattr(torch, dst) and got.shape == x.shape and torch.equal(x, keep)
    assert rel(got, oracle(x)) <= tol(5) + (BF16 if dst == 'bfloat16' else 0.0)


@pytest.mark.parametrize('kind', ['rank one', 'spikes', 'geometric', 'equal rows'])
@pytest.mark.parametrize('shape', [(2, 200, 320), (2, 320, 200), (12, 384, 1536)])
@pytest.mark.parametrize('dst', [torch.float32, torch.bfloat16])
def test_spectra_that_are_hard(kind, shape, dst):
    """Directions that are empty or tiny: roundings fall into them and are multiplied by 3.44 a step."""
    L, r, c = shape
    g = torch.Generator().manual_seed(3)
    if kind == 'rank one':
        x = torch.randn(L, r, 1, generator=g) @ torch.randn(L, 1, c, generator=g)
    elif kind == 'equal rows':
        x = torch.randn(L, 1, c, generator=g).expand(L, r, c).contiguous()
    elif kind == 'spikes':
        x = torch.randn(L, r, 3, generator=g) @ torch.randn(L, 3, c, generator=g) + 1e-4 * torch.randn(L, r, c, generator=g)
    else:
        m = min(r, c)
        u, v = (torch.linalg.qr(torch.randn(n, m, generator=g))[0] for n in (r, c))
        x = ((u * torch.logspace(0, -6, m)) @ v.T).expand(L, r, c).contiguous()
    x = x.to(DEV)
    e = rel(ops.orthogonalize(x, out_dtype=dst), oracle(x))
    print(f'{kind} {shape} {dst}: {e:.2e}')
    assert e <= tol(5) + (BF16 if dst == torch.bfloat16 else 0.0)


@pytest.mark.parametrize('steps', [1, 2, 8])
@pytest.mark.parametrize('co', [CO, (1.875, -1.25, 0.375), (1.5, -0.5, 0.0)])
def test_steps_and_coefficients(steps, co):
    x = grads(2, 70, 200)
    e = rel(ops.orthogonalize(x, steps=steps, coefficients=co), oracle(x, steps, co))
    assert e <= tol(steps), e


def test_result_is_orthogonal_with_the_convergent_polynomial():
    """(15 s - 10 s^3 + 3 s^5) / 8 has the fixed point 1 on (0, 1]: many steps give U V^T of the singular value decomposition."""
    x = grads(1, 40, 90)
    got = ops.orthogonalize(x, steps=24, coefficients=(1.875, -1.25, 0.375))[0].double().cpu()
    u, _, vh = torch.linalg.svd(x[0].double().cpu(), full_matrices=False)
    assert float((got @ got.T - torch.eye(40, dtype=torch.float64)).abs().max()) < 1e-5
    assert float((got - u @ vh).norm() / (u @ vh).norm()) < 1e-4


def test_scale_of_the_input_does_not_matter_and_zero_stays_zero():
    x = grads(1, 50, 60)
    want = ops.orthogonalize(x)
    for s in (2.0 ** 40, 2.0 ** 80):                                   # sums of squares beyond 2^127 are formed in 64 bits
        assert torch.equal(ops.orthogonalize(x * s), want)
    assert torch.equal(ops.orthogonalize(x * 2.0 ** -30, eps=1e-30), ops.orthogonalize(x, eps=1e-30))
    assert bool((ops.orthogonalize(torch.zeros(2, 30, 70, device=DEV)) == 0).all())
    small = x * (1e-9 / float(x.norm()))                               # below eps: divided by eps
    assert rel(ops.orthogonalize(small, eps=1e-7), oracle(small, eps=1e-7)) <= tol(5)


def test_non_finite_matrix_does_not_reach_its_neighbours():
    x = grads(4, 70, 90)
    want = ops.orthogonalize(x)
    for bad in (float('nan'), float('inf')):
        y = x.clone()
        y[2, 69, 3] = bad
        got = ops.orthogonalize(y)
        assert bool(got[2].isnan().all())
        assert torch.equal(got[[0, 1, 3]], want[[0, 1, 3]])


def test_views_in_place_empty_and_memory_around():
    x = grads(3, 70, 45)
    want = ops.orthogonalize(x)
    buf = torch.full((5, 76, 51), 3.0, device=DEV)
    v = buf[1:4, 2:72, 3:48]                                           # stride, pitch and start that are no multiple of 4 elements
    v.copy_(x)
    assert torch.equal(ops.orthogonalize(v), want)
    assert torch.equal(ops.orthogonalize(v, out=v), want)
    v.fill_(3.0)
    assert bool((buf == 3.0).all())
    one = ops.orthogonalize(x[0, ::2])                                 # every other row of one matrix
    assert torch.equal(one, ops.orthogonalize(x[0, ::2].contiguous()))
    for shape in ((0, 5, 6), (2, 0, 6), (2, 5, 0)):
        assert ops.orthogonalize(torch.empty(shape, device=DEV)).shape == shape


def muon_oracle(p, g, m, hyper, nesterov, scale, steps=5):
    lr, mu, wd, gs = [float(v) for v in hyper.double()]
    g = g.double() * gs
    m = mu * m.double() + (1 - mu) * g
    u = (1 - mu) * g + mu * m if nesterov else m
    three = u if u.dim() == 3 else u[None]
    o = oracle(three, steps)
    o = o if u.dim() == 3 else o[0]
    return p.double() * (1 - lr * wd) - lr * scale * o, m, o


def check_muon(p0, g0, m0, p, m, hyper, nesterov, scale):
    rp, rm, o = muon_oracle(p0, g0, m0, hyper, nesterov, scale)
    lr, mu, wd, gs = [float(v) for v in hyper.double()]
    # momentum: three roundings of fp32
    assert bool(((m.double() - rm).abs() <= 3 * 2.0 ** -24 * (m0.double().abs() + (g0.double() * gs).abs())).all())
    # the direction is rounded before the products (relative 2^-22); parameters: four roundings, and the update's own error (2-norm)
    step = lr * scale * float(o.norm())
    err = (p.double() - rp).norm()
    assert float(err) <= 4 * 2.0 ** -24 * float(p0.double().norm() + step) + step * tol(5)


@pytest.mark.parametrize('nesterov', [True, False])
@pytest.mark.parametrize('scale', ['original', 'match_rms_adamw', 0.3])
def test_muon_step_over_mixed_stacks(nesterov, scale):
    shapes = [(2, 192, 64), (2, 64, 64), (64, 33), (1, 7, 300), (3, 256, 64), (0, 4, 4), (5, 1)]
    g = torch.Generator().manual_seed(0)
    mk = lambda s, k: (torch.randn(*s, generator=g) * k).to(DEV)
    p, gr, m = [mk(s, 0.02) for s in shapes], [mk(s, 1e-3) for s in shapes], [mk(s, 1e-3) for s in shapes]
    hyper = torch.tensor([2e-3, 0.9, 0.1, 0.5], device=DEV)
    p0, m0, g0 = [t.clone() for t in p], [t.clone() for t in m], [t.clone() for t in gr]
    ops.muon_step(p, gr, m, hyper, nesterov=nesterov, scale=scale)
    for i, s in enumerate(shapes):
        if 0 in s:
            continue
        assert torch.equal(gr[i], g0[i])
        check_muon(p0[i], g0[i], m0[i], p[i], m[i], hyper, nesterov, ops.muon_scale(scale, s[-2], s[-1]))


def test_muon_step_with_large_tiles():
    """wide, tall and square stacks of one 384-wide model in one step (128 x 128 tiles)"""
    shapes = [(6, 1152, 384), (6, 384, 384), (6, 1536, 384), (6, 384, 1536), (1, 380, 1530)]
    g = torch.Generator(device=DEV).manual_seed(0)
    p, gr, m = [[torch.randn(*s, generator=g, device=DEV) * k for s in shapes] for k in (0.02, 1e-3, 1e-3)]
    hyper = torch.tensor([2e-3, 0.95, 0.1, 1.0], device=DEV)
    p0, m0 = [t.clone() for t in p], [t.clone() for t in m]
    ops.muon_step(p, gr, m, hyper)
    for i, s in enumerate(shapes):
        check_muon(p0[i], gr[i], m0[i], p[i], m[i], hyper, True, ops.muon_scale('original', *s[1:]))


def test_muon_many_items_and_bitwise_repeat():
    """more stacks than one launch takes; the same step twice gives the same bits"""
    shapes = [(16 + 5 * i, 90 - 3 * i) for i in range(20)]
    g = torch.Generator().manual_seed(0)
    p0, g0, m0 = [[(torch.randn(*s, generator=g) * k).to(DEV) for s in shapes] for k in (0.02, 1e-3, 1e-3)]
    hyper = torch.tensor([1e-2, 0.95, 0.0, 1.0], device=DEV)
    res = []
    for _ in range(2):
        p, m = [t.clone() for t in p0], [t.clone() for t in m0]
        ops.muon_step(p, g0, m, hyper)
        res.append((p, m))
    for i, s in enumerate(shapes):
        check_muon(p0[i], g0[i], m0[i], res[0][0][i], res[0][1][i], hyper, True, ops.muon_scale('original', *s))
        assert torch.equal(res[0][0][i], res[1][0][i]) and torch.equal(res[0][1][i], res[1][1][i])


def test_muon_planes_zero_grad_and_memory_around():
    L, r, c = 3, 50, 70
    g = torch.Generator().manual_seed(2)
    buf = {k: torch.full((L, r * c + 40), 5.0, device=DEV) for k in 'pgm'}
    pl = [torch.full((L, r * c + 40), 5.0, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
    view = lambda t: t[:, 8:8 + r * c].unflatten(1, (r, c))
    init = {k: (torch.randn(L, r, c, generator=g) * 0.01).to(DEV) for k in 'pgm'}
    for k in 'pgm':
        view(buf[k]).copy_(init[k])
    hyper = torch.tensor([1e-2, 0.95, 0.01, 1.0], device=DEV)
    ops.muon_step([view(buf['p'])], [view(buf['g'])], [view(buf['m'])], hyper, planes=[(view(pl[0]), view(pl[1]))], zero_grad=True)
    check_muon(init['p'], init['g'], init['m'], view(buf['p']), view(buf['m']), hyper, True, 1.0)
    assert bool((view(buf['g']) == 0).all())
    p = view(buf['p'])
    assert torch.equal(view(pl[0]), p.to(torch.bfloat16))
    assert torch.equal(view(pl[1]), (p - view(pl[0]).float()).to(torch.bfloat16))
    for t in list(buf.values()) + pl:
        view(t).fill_(5.0)
        assert bool((t == 5.0).all())


def test_muon_agrees_with_the_plain_optimizer_rule_over_steps():
    """Ten steps against the 64-bit rule run beside it on its own state: errors do not build up beyond ten single steps'."""
    g = torch.Generator().manual_seed(4)
    p = (torch.randn(48, 80, generator=g) * 0.05).to(DEV)
    m = torch.zeros_like(p)
    hyper = torch.tensor([1e-2, 0.95, 0.01, 1.0], device=DEV)
    rp, rm = p.double(), m.double()
    scale = ops.muon_scale('original', 48, 80)
    for k in range(10):
        gr = (torch.randn(48, 80, generator=g) * 1e-3).to(DEV)
        ops.muon_step([p], [gr], [m], hyper)
        rp, rm, _ = muon_oracle(rp, gr, rm, hyper, True, scale)
    step = float(hyper[0]) * scale * 48 ** 0.5
    assert float((p.double() - rp).norm()) <= 10 * (4 * 2.0 ** -24 * float(rp.norm()) + step * 2 * tol(5))


def test_on_another_stream_and_in_two_replayed_graphs():
    x = grads(2, 100, 150)
    want = ops.orthogonalize(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.orthogonalize(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # two captured steps, replayed in turn with eager work between: each follows its inputs and the schedule in hyper
    g = torch.Generator().manual_seed(1)
    mk = lambda r, c: [(torch.randn(r, c, generator=g) * 0.02).to(DEV) for _ in range(3)]
    state = [mk(90, 70), mk(33, 200)]
    hyper = torch.tensor([1e-2, 0.95, 0.01, 1.0], device=DEV)
    eager = [[t.clone() for t in s] for s in state]
    graphs = []
    for p, gr, m in state:
        keep = p.clone(), m.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.muon_step([p], [gr], [m], hyper)
        p.copy_(keep[0]), m.copy_(keep[1])
        graphs.append(graph)
    for k in range(4):
        hyper[0] = 1e-2 / (k + 1)
        for s, e, graph in zip(state, eager, graphs):
            s[1].mul_(-1.5), e[1].mul_(-1.5)
            graph.replay()
            ops.muon_step([e[0]], [e[1]], [e[2]], hyper)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(s, e)), k


def test_two_streams_at_once():
    """two calls that overlap in time: each has its own workspace"""
    xs = [grads(4, 300, 500, seed=s) for s in (1, 2)]
    want = [ops.orthogonalize(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = ops.orthogonalize(xs[i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_column_blocks_and_row_blocks_of_one_matrix():
    """Parameters that are blocks of one tensor (their address ranges interleave, their elements do not): the step of separate tensors, bit for bit."""
    hyper = torch.tensor([0.02, 0.9, 0.1, 1.0], device=DEV)
    full = [grads(3, 300, 200, seed=s) for s in range(3)]
    cut = lambda t: [t[:, :120, :64], t[:, :120, 64:200], t[:, 120:300, :], ]
    cols = lambda t: [t[0, :, :64], t[0, :, 64:70], t[0, :, 70:]]                # count 1
    for blocks in (cut, cols):
        apart = [[v.contiguous().clone() for v in blocks(t)] for t in full]
        both = [t.clone() for t in full]
        ops.muon_step(*apart, hyper, zero_grad=True)
        ops.muon_step(*[blocks(t) for t in both], hyper, zero_grad=True)
        for t, parts in zip(both, apart):
            for v, w in zip(blocks(t), parts):
                assert torch.equal(v, w)
        if blocks is cols:
            for t, f in zip((both[0], both[2]), (full[0], full[2])):
                assert torch.equal(t[1:], f[1:])                                 # rows behind the last block are left alone


def test_shared_parameters_are_refused():
    p, g, m = (grads(2, 40, 30, seed=s) for s in range(3))
    hyper = torch.tensor([0.02, 0.9, 0.1, 1.0], device=DEV)
    keep = [t.clone() for t in (p, g, m)]
    for args in (([p, p], [g, g], [m, m]), ([p, p[1]], [g, g[1]], [m, m[1]]), ([p], [g], [g]), ([p[0], p[1]], [g[0], g[1]], [m[0], m[0]])):
        with pytest.raises(RuntimeError, match='shares memory'):
            ops.muon_step(*args, hyper)
    assert all(torch.equal(a, b) for a, b in zip(keep, (p, g, m)))


@pytest.mark.parametrize('shapes', [[(1, 192, 192)], [(2, 64, 300), (1, 300, 60)], [(3, 128, 200), (2, 210, 100)], [(1, 150, 700), (1, 700, 190), (2, 30, 90)]])
@pytest.mark.parametrize('zero', [False, True])
def test_muon_step_over_small_sides(shapes, zero):
    """smaller sides of one, two and three tiles, wide and tall, apart and mixed: polynomial and product in one launch"""
    g = torch.Generator().manual_seed(1)
    p, gr, m = [[(torch.randn(*s, generator=g) * k).to(DEV) for s in shapes] for k in (0.02, 1e-3, 1e-3)]
    planes = [tuple(torch.zeros(*s, dtype=torch.bfloat16, device=DEV) for _ in range(2)) for s in shapes]
    hyper = torch.tensor([2e-3, 0.95, 0.1, 1.0], device=DEV)
    p0, m0, g0 = [t.clone() for t in p], [t.clone() for t in m], [t.clone() for t in gr]
    ops.muon_step(p, gr, m, hyper, planes=planes, zero_grad=zero)
    for i, s in enumerate(shapes):
        check_muon(p0[i], g0[i], m0[i], p[i], m[i], hyper, True, ops.muon_scale('original', *s[1:]))
        hi = p[i].bfloat16()
        assert torch.equal(planes[i][0], hi) and torch.equal(planes[i][1], (p[i] - hi.float()).bfloat16())
        assert torch.equal(gr[i], torch.zeros_like(gr[i]) if zero else g0[i])


def test_stacks_whose_offsets_pass_32_bits():
    """matrices 1.2 10^9 elements apart, and a workspace of more than 2^32 bytes: the results of compact stacks, bit for bit"""
    stride, r, c = 1_200_000_000, 70, 150
    buf = torch.empty(2 * stride + r * c, device=DEV)
    far = buf.as_strided((3, r, c), (stride, c, 1))
    g, m, p = (grads(3, r, c, seed=s) for s in range(3))
    far.copy_(p)
    hyper = torch.tensor([0.02, 0.9, 0.1, 1.0], device=DEV)
    m2 = m.clone()
    ops.muon_step([far], [g], [m2], hyper)
    ops.muon_step([p], [g], [m], hyper)
    assert torch.equal(far, p) and torch.equal(m, m2)
    far.copy_(g)
    assert torch.equal(ops.orthogonalize(far, out=far), ops.orthogonalize(g))
    del buf, far
    many = grads(1, 192, 192).expand(20000, 192, 192)
    out = ops.orthogonalize(many)
    few = ops.orthogonalize(many[:40].contiguous())                  # (fewer matrices take other tiles: the tolerance of two results)
    assert torch.equal(out[0], out[-1]) and torch.equal(out[0], out[9999])
    assert rel(out[-1:], few[:1]) <= 2 * tol(5)
