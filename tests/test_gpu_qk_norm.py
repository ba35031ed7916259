"""Head norm + position rotation (s3d_qk_norm_rope_fwd / _bwd) against the formulas in 64 bits, and against differences."""
import pytest
import torch

from simple3d_former_amd import ops

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
EPS = 1e-6


def make(rows, H, Hkv, hd, pair, seed=0, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, (H + 2 * Hkv) * hd, generator=g) * scale).to(DEV)
    hi = x.to(torch.bfloat16)
    return hi, ((x - hi.float()).to(torch.bfloat16) if pair else None)


def whole(hi, lo):
    return hi.double() + lo.double() if lo is not None else hi.double()


def gains(hd, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [(1 + 0.2 * torch.randn(hd, generator=g)).to(DEV) for _ in range(2)]


def table(T, hd, seed=5):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand(T, hd // 2, generator=g, dtype=torch.float64) * 6.28
    return a.cos().float().to(DEV), a.sin().float().to(DEV)


def angles(rope, index):
    """cos, sin [rows, 1, hd/2] in 64 bits; index [rows], anything outside the table = no rotation"""
    cos, sin = rope[0].double(), rope[1].double()
    on = ((index >= 0) & (index < cos.shape[0]))[:, None]
    i = index.clamp(0, cos.shape[0] - 1).long()
    return torch.where(on, cos[i], 1.0)[:, None], torch.where(on, sin[i], 0.0)[:, None]


def oracle(x, H, Hkv, hd, gq, gk, cs, inter):
    """out [rows, W] in 64 bits and the size of the terms each output is a sum of (for the tolerance)"""
    x = x.view(x.shape[0], -1, hd)

    def one(t, g):
        z = t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS)
        z = z if g is None else z * g.double()
        if cs is None:
            return z, z.abs()
        c, s = cs
        a, b = (z[..., 0::2], z[..., 1::2]) if inter else (z[..., :hd // 2], z[..., hd // 2:])
        y = (a * c - b * s, b * c + a * s)
        m = (a.abs() + b.abs(),) * 2
        if inter:
            return torch.stack(y, -1).flatten(-2), torch.stack(m, -1).flatten(-2)
        return torch.cat(y, -1), torch.cat(m, -1)
    q, mq = one(x[:, :H], gq)
    k, mk = one(x[:, H:H + Hkv], gk)
    v = x[:, H + Hkv:]
    return torch.cat([q, k, v], 1).flatten(1), torch.cat([mq, mk, v.abs()], 1).flatten(1)


SHAPES = [(1, 6, 6, 64, False), (1, 1, 1, 16, True), (26, 6, 6, 64, True), (257, 3, 3, 256, False), (33, 3, 3, 192, True), (1031, 6, 2, 80, False),
          (70, 5, 1, 48, True), (9, 2, 2, 32, False), (513, 12, 4, 128, False), (40000, 3, 3, 64, False), (5, 1, 3, 240, True)]


@pytest.mark.parametrize('rows,H,Hkv,hd,pair', SHAPES)
@pytest.mark.parametrize('inter', [False, True])
@pytest.mark.parametrize('rot', ['none', 'index', 'pos'])
def test_forward(rows, H, Hkv, hd, pair, inter, rot):
    hi, lo = make(rows, H, Hkv, hd, pair)
    gq, gk = gains(hd) if rot != 'none' else (None, None)
    T = 23
    rope = None if rot == 'none' else table(T, hd)
    pos, st, cs = None, 1, None
    if rot == 'pos':
        pos = torch.randint(-2, T + 2, (rows,), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(DEV)
        cs = angles(rope, pos)
    elif rot == 'index':
        st = 3
        cs = angles(rope, (torch.arange(rows, device=DEV) // st) % T)
    ohi, olo = ops.qk_norm_rope_fwd(hi, lo, H, hd, Hkv=Hkv, q_gain=gq, k_gain=gk, rope=rope, pos=pos, st=st, eps=EPS, interleaved=inter)
    assert (olo is None) == (lo is None)
    ref, mag = oracle(whole(hi, lo), H, Hkv, hd, gq, gk, cs, inter)
    # one rounding to bf16 (2^-8 of the value; a pair 2^-16), under it fp32: about 30 roundings of the mean, the gain and the rotation
    tol = ref.abs() * (2.0 ** -16 if pair else 2.0 ** -8) + 32 * 2.0 ** -24 * mag + 1e-30
    assert bool(((whole(ohi, olo) - ref).abs() <= tol).all())
    W = (H + Hkv) * hd
    assert torch.equal(ohi[:, W:], hi[:, W:]) and (lo is None or torch.equal(olo[:, W:], lo[:, W:]))        # values: copied bit for bit


@pytest.mark.parametrize('rows,H,Hkv,hd,pair', SHAPES)
@pytest.mark.parametrize('inter,gain', [(False, True), (True, False)])
def test_backward(rows, H, Hkv, hd, pair, inter, gain):
    hi, lo = make(rows, H, Hkv, hd, pair)
    dhi, dlo = make(rows, H, Hkv, hd, pair, seed=9, scale=0.03)
    gq, gk = gains(hd) if gain else (None, None)
    T = 19
    rope = table(T, hd)
    pos = torch.randint(-2, T + 2, (rows,), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(DEV)
    kw = dict(Hkv=Hkv, q_gain=gq, k_gain=gk, rope=rope, pos=pos, eps=EPS, interleaved=inter)
    ghi, glo, dgq, dgk = ops.qk_norm_rope_bwd(dhi, dlo, hi, lo, H, hd, **kw)
    x = whole(hi, lo).requires_grad_()
    oq, ok = (torch.ones(hd, device=DEV, dtype=torch.float64) if g is None else g.double() for g in (gq, gk))
    oq.requires_grad_(), ok.requires_grad_()
    cs = angles(rope, pos)
    y, _ = oracle(x, H, Hkv, hd, oq, ok, cs, inter)
    rx, rq, rk = torch.autograd.grad(y, [x, oq, ok], whole(dhi, dlo))
    # size of what dx is the difference of: r (|d| + |x r| mean|d x r|), |d| <= |R^T dy| gain
    xv, dv = whole(hi, lo).view(rows, -1, hd), whole(dhi, dlo).abs().view(rows, -1, hd)
    r = 1 / torch.sqrt((xv * xv).mean(-1, keepdim=True) + EPS)
    gmax = max(float(oq.abs().max()), float(ok.abs().max()))
    big = gmax * (dv[..., 0::2] + dv[..., 1::2]).repeat_interleave(2, -1) if inter else gmax * (dv[..., :hd // 2] + dv[..., hd // 2:]).repeat(1, 1, 2)
    mag = (r * (big + (xv * r).abs() * (big * (xv * r).abs()).mean(-1, keepdim=True))).flatten(1)
    tol = rx.abs() * (2.0 ** -16 if pair else 2.0 ** -8) + 64 * 2.0 ** -24 * mag + 1e-30
    got = whole(ghi, glo)
    W = (H + Hkv) * hd
    assert bool(((got - rx).abs() <= tol)[:, :W].all())
    assert torch.equal(ghi[:, W:], dhi[:, W:]) and (dlo is None or torch.equal(glo[:, W:], dlo[:, W:]))
    # gains: a sum over rows and heads of products with about 12 roundings each, added 16 .. 80 at a time in fp32, then in 64 bits
    t = (big / gmax * (xv * r).abs())
    for got1, ref1, part in ((dgq, rq, t[:, :H]), (dgk, rk, t[:, H:H + Hkv])):
        assert bool(((got1.double() - ref1).abs() <= 2.0 ** -24 * 128 * part.sum((0, 1)) + 1e-30).all())


def test_backward_against_differences():
    """d(sum out * w) / d(direction) from two evaluations of the 64-bit forward at +- h: independent of autograd's formulas."""
    rows, H, Hkv, hd = 17, 2, 1, 32
    hi, _ = make(rows, H, Hkv, hd, False)
    w, _ = make(rows, H, Hkv, hd, False, seed=4, scale=0.1)
    gq, gk = gains(hd)
    rope = table(rows, hd)
    cs = angles(rope, torch.arange(rows, device=DEV))
    dx, _, dgq, dgk = ops.qk_norm_rope_bwd(w, None, hi, None, H, hd, Hkv=Hkv, q_gain=gq, k_gain=gk, rope=rope, eps=EPS)
    g = torch.Generator().manual_seed(8)
    vx = torch.randn(hi.shape, generator=g, dtype=torch.float64).to(DEV)
    vq, vk = (torch.randn(hd, generator=g, dtype=torch.float64).to(DEV) for _ in range(2))
    h = 1e-5

    def f(t):
        y, _ = oracle(hi.double() + t * vx, H, Hkv, hd, gq.double() + t * vq, gk.double() + t * vk, cs, False)
        return float((y * w.double()).sum())
    want = (f(h) - f(-h)) / (2 * h)
    got = float((dx.double() * vx).sum() + (dgq.double() * vq).sum() + (dgk.double() * vk).sum())
    # dx is rounded to bf16: independent errors of at most 2^-8 |dx| against vx
    tol = 4 * 2.0 ** -8 * float((dx.double() * vx).square().sum().sqrt()) + 1e-4 * abs(want)
    assert abs(got - want) <= tol, (got, want, tol)


def test_strided_rows_in_place_and_memory_around():
    rows, H, hd = 37, 3, 64
    W = 3 * H * hd
    hi, lo = make(rows, H, H, hd, True)
    rope = table(rows, hd)
    want = ops.qk_norm_rope_fwd(hi, lo, H, hd, rope=rope)
    buf = torch.full((2, rows + 4, W + 24), 7.0, dtype=torch.bfloat16, device=DEV)
    v = buf[:, 2:2 + rows, 8:8 + W]
    v[0].copy_(hi), v[1].copy_(lo)
    got = ops.qk_norm_rope_fwd(v[0], v[1], H, hd, rope=rope, out=(v[0], v[1]))                  # in place, pitch W + 24
    assert got[0].data_ptr() == v[0].data_ptr()
    assert torch.equal(v[0], want[0]) and torch.equal(v[1], want[1])
    v.fill_(7.0)
    assert bool((buf == 7.0).all())                                                             # nothing outside the rows was touched
    # backward: dqkv over dout
    dhi, dlo = make(rows, H, H, hd, True, seed=2)
    want = ops.qk_norm_rope_bwd(dhi, dlo, hi, lo, H, hd, rope=rope)
    v[0].copy_(dhi), v[1].copy_(dlo)
    got = ops.qk_norm_rope_bwd(v[0], v[1], hi, lo, H, hd, rope=rope, out=(v[0], v[1]))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    v.fill_(7.0)
    assert bool((buf == 7.0).all())


def test_pairs_and_plain_planes_mixed():
    """A pair into one plane and one plane into a pair, forward and backward: the same values as with the planes alike."""
    rows, H, hd = 21, 2, 64
    hi, lo = make(rows, H, H, hd, True)
    d, dlo = make(rows, H, H, hd, True, seed=1)
    rope = table(rows, hd)
    new = lambda: torch.empty_like(hi)
    pair = ops.qk_norm_rope_fwd(hi, lo, H, hd, rope=rope)
    one, none = ops.qk_norm_rope_fwd(hi, lo, H, hd, rope=rope, out=(new(), None))
    V = 2 * H * hd                                                       # queries and keys: the hi plane is the value rounded to bf16.  Values: the
    assert none is None and torch.equal(one[:, :V], pair[0][:, :V])      # planes bit for bit, or their sum rounded (not hi where lo is half a step)
    assert torch.equal(one[:, V:], (hi.float() + lo.float()).to(torch.bfloat16)[:, V:])
    a, b = ops.qk_norm_rope_fwd(hi, None, H, hd, rope=rope, out=(new(), new()))
    ref, mag = oracle(hi.double(), H, H, hd, None, None, angles(rope, torch.arange(rows, device=DEV)), False)
    assert bool(((whole(a, b) - ref).abs() <= ref.abs() * 2.0 ** -16 + 32 * 2.0 ** -24 * mag).all())
    assert bool((b[:, V:] == 0).all()) and torch.equal(a[:, V:], hi[:, V:])
    full = ops.qk_norm_rope_bwd(d, dlo, hi, lo, H, hd, rope=rope)
    one = ops.qk_norm_rope_bwd(d, dlo, hi, lo, H, hd, rope=rope, out=(new(), None))
    assert torch.equal(one[0][:, :V], full[0][:, :V]) and torch.equal(one[2], full[2]) and torch.equal(one[3], full[3])
    full = ops.qk_norm_rope_bwd(d, None, hi, lo, H, hd, rope=rope, out=(new(), new()))
    one = ops.qk_norm_rope_bwd(d, None, hi, lo, H, hd, rope=rope)
    assert one[1] is None and torch.equal(one[0], full[0]) and bool((full[1][:, V:] == 0).all())


def test_zero_rows_no_rows_and_special_values():
    H, hd = 2, 48
    W = 3 * H * hd
    hi, _ = make(6, H, H, hd, False)
    hi[2] = 0
    hi[4, 5] = float('nan')
    out, _ = ops.qk_norm_rope_fwd(hi, None, H, hd)
    assert bool((out[2] == 0).all())                                                    # a zero head stays zero
    assert bool(out[4, :hd].isnan().all()) and bool(out[4, hd:].isfinite().all())       # a NaN stays in its head
    assert bool(out[[0, 1, 2, 3, 5]].isfinite().all())
    empty = torch.empty(0, W, dtype=torch.bfloat16, device=DEV)
    assert ops.qk_norm_rope_fwd(empty, None, H, hd)[0].shape == (0, W)
    _, _, dq, dk = ops.qk_norm_rope_bwd(empty, None, empty, None, H, hd)
    assert bool((dq == 0).all()) and bool((dk == 0).all())
    # a NaN in a query's gradient stays out of the keys' gains
    hi, _ = make(6, H, H, hd, False)
    d, _ = make(6, H, H, hd, False, seed=1)
    d[3, 0] = float('nan')
    _, _, dq, dk = ops.qk_norm_rope_bwd(d, None, hi, None, H, hd)
    assert bool(dq.isnan().any()) and bool(dk.isfinite().all())


def test_gain_gradients_accumulate_and_repeat_bitwise():
    rows, H, hd = 3000, 3, 64
    hi, _ = make(rows, H, H, hd, False)
    d, _ = make(rows, H, H, hd, False, seed=1)
    rope = table(rows, hd)
    a = ops.qk_norm_rope_bwd(d, None, hi, None, H, hd, rope=rope)
    b = ops.qk_norm_rope_bwd(d, None, hi, None, H, hd, rope=rope)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2]) and torch.equal(a[3], b[3])
    base = torch.ones(2, hd, device=DEV)
    ops.qk_norm_rope_bwd(d, None, hi, None, H, hd, rope=rope, gain_grads=(base[0], base[1]))
    assert torch.equal(base[0], 1 + a[2]) and torch.equal(base[1], 1 + a[3])


def test_on_another_stream_and_in_a_replayed_graph():
    rows, H, hd = 900, 3, 64
    hi, _ = make(rows, H, H, hd, False)
    d, _ = make(rows, H, H, hd, False, seed=1)
    gq, gk = gains(hd)
    rope = table(rows, hd)
    kw = dict(q_gain=gq, k_gain=gk, rope=rope)
    sx, sd = hi.clone(), d.clone()

    def both():
        o, _ = ops.qk_norm_rope_fwd(sx, None, H, hd, **kw)
        return (o,) + tuple(t for t in ops.qk_norm_rope_bwd(sd, None, sx, None, H, hd, **kw) if t is not None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    want = both()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for k in range(4):
        sx.copy_(hi * (k + 1))
        sd.copy_(d.roll(k, 0))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, both())), k


def test_rope_table_axes_and_far_positions():
    cos, sin = ops.rope_table(torch.tensor([0, 1, 10 ** 7]), 32)
    f = 10000.0 ** (-torch.arange(16, dtype=torch.float64) / 16)
    ang = 1e7 * f
    assert torch.equal(cos[2], ang.cos().float()) and torch.equal(sin[2], ang.sin().float())
    cos, sin = ops.rope_table(torch.tensor([[1, 2, 3]]), 64)            # 32 pairs: 10 for each axis, two not rotated
    assert cos.shape == (1, 32) and bool((cos[0, 30:] == 1).all()) and bool((sin[0, 30:] == 0).all())
    assert abs(float(sin[0, 10]) - torch.sin(torch.tensor(2.0)).item()) < 1e-7


def test_offsets_past_32_bits():
    """2.3 10^9 elements per plane: the last rows and the last value heads, against the same rows in a tensor of their own."""
    H, hd, rows = 6, 64, 2_000_003
    W = 3 * H * hd
    x = torch.empty(rows, W, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(5))
    gain = torch.rand(hd, device=DEV) + 0.5
    rope = tuple(t.to(DEV) for t in ops.rope_table(torch.arange(1000), hd))
    pos = (torch.arange(rows, device=DEV) % 1000).int()
    out, _ = ops.qk_norm_rope_fwd(x, None, H, hd, q_gain=gain, k_gain=gain, rope=rope, pos=pos)
    dx, _, dq, dk = ops.qk_norm_rope_bwd(out, None, x, None, H, hd, q_gain=gain, k_gain=gain, rope=rope, pos=pos)
    for s in (slice(0, 700), slice(rows // 2, rows // 2 + 700), slice(rows - 700, rows)):
        small, _ = ops.qk_norm_rope_fwd(x[s].clone(), None, H, hd, q_gain=gain, k_gain=gain, rope=rope, pos=pos[s].clone())
        assert torch.equal(out[s], small)
        back = ops.qk_norm_rope_bwd(small, None, x[s].clone(), None, H, hd, q_gain=gain, k_gain=gain, rope=rope, pos=pos[s].clone())[0]
        assert torch.equal(dx[s], back)
    assert bool(torch.isfinite(dq).all()) and bool(torch.isfinite(dk).all())


def test_one_gradient_tensor_for_both_gains_is_refused():
    x = torch.randn(20, 3 * 64, device=DEV).bfloat16()
    d = torch.zeros(64, device=DEV)
    with pytest.raises(RuntimeError, match='overlap'):
        ops.qk_norm_rope_bwd(x.clone(), None, x, None, 1, 64, gain_grads=(d, d))
    with pytest.raises(RuntimeError, match='overlap'):
        ops.qk_norm_rope_fwd(x[1:], None, 1, 64, out=(x[:-1], None))
    assert not bool(d.any())
