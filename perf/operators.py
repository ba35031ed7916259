"""What the framework's operators for normalised, rotated queries and keys and for orthogonalised updates are measured on.

qk     one pass between the qkv product and the attention of a transformer block: every query and key head is divided by its root mean
       square, scaled by a gain, and rotated by its token's position; the values pass through.  Forward and backward.
ortho  a stack of matrices through the Newton-Schulz products X <- a X + (b A + c A^2) X, A = X X^T.
muon   the optimizer step over several stacks of weight matrices: momentum, the orthogonalised update, decoupled decay."""
import math

import torch

own = False

COEFF = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-6          # inside the root mean square
NORM_EPS = 1e-7     # smallest norm a matrix is divided by


def listed():
    return [
        # one voxel grid through a 384-wide encoder (26 tokens, 6 heads): evaluation of a single sample, the call's latency
        dict(name='qk one grid', op='qk', back=False, B=1, N=26, H=6, Hkv=6, hd=64, pair=False, inter=False, pos=False, gains=True),
        # the benchmark's training step (64 grids of 26 tokens) in the split-bf16 forward: every tensor a pair of planes
        dict(name='qk grids pair', op='qk', back=False, B=64, N=26, H=6, Hkv=6, hd=64, pair=True, inter=False, pos=True, gains=True),
        # first pass of the grouped 128^3 model: 64 x 196 groups of 15 tokens, 3 heads of 256
        dict(name='qk groups', op='qk', back=False, B=12544, N=15, H=3, Hkv=3, hd=256, pair=False, inter=False, pos=False, gains=True),
        # backward of a part-segmentation step: 32 clouds of 513 tokens, 3 heads of 64
        dict(name='qk clouds back', op='qk', back=True, B=32, N=513, H=3, Hkv=3, hd=64, pair=False, inter=False, pos=True, gains=True),
        # backward of the grouped model's first pass: the largest
        dict(name='qk groups back', op='qk', back=True, B=12544, N=15, H=3, Hkv=3, hd=256, pair=False, inter=False, pos=False, gains=True),
        # odd sizes, shared key heads, neighbouring pairs
        dict(name='qk odd back', op='qk', back=True, B=7, N=1031, H=6, Hkv=2, hd=80, pair=False, inter=True, pos=True, gains=True),
        # one 192 x 192 projection: the smallest matrix of the configurations, a chain of 15 small products
        dict(name='ortho one', op='ortho', L=1, r=192, c=192, src='float32', dst='bfloat16'),
        # the twelve first MLP weights of the 384-wide model (tall: rows > cols), kept in 32 bits
        dict(name='ortho mlp', op='ortho', L=12, r=1536, c=384, src='float32', dst='float32'),
        # a few large square matrices of bf16 gradients: the largest products
        dict(name='ortho large', op='ortho', L=4, r=2048, c=2048, src='bfloat16', dst='bfloat16'),
        # one 192-wide transformer block: qkv, proj, fc1, fc2
        dict(name='muon block', op='muon', L=1, D=192, odd=0, nesterov=True),
        # the block weights of the 384-wide model, twelve blocks: the ordinary optimizer step
        dict(name='muon model', op='muon', L=12, D=384, odd=0, nesterov=True),
        # sides that are no multiple of any tile
        dict(name='muon odd', op='muon', L=3, D=250, odd=37, nesterov=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(('qk', 'qk', 'ortho', 'muon'))
    if op == 'qk':
        hd = rng.choice((16, 32, 48, 64, 80, 96, 128, 192, 256))
        Hkv = rng.randint(1, 6)
        H = Hkv * rng.choice((1, 1, 1, 2, 3))
        N = _log(rng, 1, 2049)
        most = 12544 * 15 * 9 * 256 // ((H + 2 * Hkv) * hd * N)
        back, pair = rng.random() < 0.5, rng.random() < 0.25
        return dict(op='qk', back=back, B=_log(rng, 1, max(1, min(4096, most // 4))), N=N, H=H, Hkv=Hkv, hd=hd, pair=pair,
                    inter=rng.random() < 0.3, pos=rng.random() < 0.5, gains=rng.random() < 0.8)
    if op == 'ortho':
        r, c = _log(rng, 16, 1600), _log(rng, 16, 1600)
        src, dst = rng.choice((('float32', 'float32'), ('float32', 'bfloat16'), ('bfloat16', 'bfloat16')))
        return dict(op='ortho', L=rng.randint(1, 6), r=r, c=c, src=src, dst=dst)
    return dict(op='muon', L=rng.randint(1, 12), D=_log(rng, 24, 384), odd=rng.choice((0, 0, rng.randint(1, 60))), nesterov=rng.random() < 0.7)


def _muon_shapes(case):
    D, o = case['D'], case['odd']
    return [(3 * D + o, D), (D, D), (4 * D, D + o), (D, 4 * D + o)]


# ------------------------------------------------------------------------------------------------ inputs
def _gradients(g, L, r, c):
    """What momentum and gradients of a weight look like: noise and a few strong directions."""
    dev = g.device
    noise = torch.randn(L, r, c, generator=g, device=dev)
    u = torch.randn(L, r, 8, generator=g, device=dev)
    v = torch.randn(L, 8, c, generator=g, device=dev)
    return (noise + 0.25 * torch.bmm(u, v)) * 1e-3


def _table(T, hd, axis):
    """cos / sin of the rotation angles of T positions: three axes of a grid (8 cells a side) or one running index; angles in 64 bits.
    Pairs that the axes do not fill are not rotated."""
    half = hd // 2
    t = torch.arange(T, dtype=torch.float64)
    co = torch.stack([torch.remainder(t, 8), torch.remainder(torch.floor(t / 8), 8), torch.floor(t / 64)], 1) if axis == 3 else t[:, None]
    per = half // axis
    f = 10000.0 ** (-torch.arange(per, dtype=torch.float64) / max(per, 1))
    ang = torch.zeros(T, half, dtype=torch.float64)
    ang[:, :per * axis] = (co[:, :, None] * f).reshape(T, per * axis)
    return torch.cos(ang).float(), torch.sin(ang).float()


def prepare(case, seed):
    dev = torch.device('cuda' if torch.cuda.is_available() else 'cpu')
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    s = dict(case=case)
    if case['op'] == 'qk':
        rows, hd, H, Hkv = case['B'] * case['N'], case['hd'], case['H'], case['Hkv']
        W = (H + 2 * Hkv) * hd

        def planes(scale):
            x = torch.randn(rows, W, generator=g, device=dev) * scale
            hi = x.to(torch.bfloat16)
            return torch.stack([hi, (x - hi.float()).to(torch.bfloat16)]) if case['pair'] else hi[None].contiguous()
        s['qkv'] = planes(1.5)
        cos, sin = _table(case['N'], hd, 3 if hd >= 48 else 1)
        s['cos'], s['sin'] = cos.to(dev), sin.to(dev)
        s['pos'] = None
        if case['pos']:     # the first token of a sequence is the class token (no position); the others are shuffled positions
            p = torch.randint(0, case['N'], (case['B'], case['N']), generator=g, device=dev, dtype=torch.int32)
            p[:, 0] = -1
            s['pos'] = p.reshape(-1).contiguous()
        s['gq'] = 1 + 0.1 * torch.randn(hd, generator=g, device=dev) if case['gains'] else None
        s['gk'] = 1 + 0.1 * torch.randn(hd, generator=g, device=dev) if case['gains'] else None
        if case['back']:
            s['dout'] = planes(0.01)
    elif case['op'] == 'ortho':
        s['x'] = _gradients(g, case['L'], case['r'], case['c']).to(getattr(torch, case['src']))
    else:
        s['hyper'] = torch.tensor([1e-3, 0.95, 0.05, 1.0], device=dev)      # learning rate, momentum, decay, gradient scale
        s['p'] = [torch.randn(case['L'], r, c, generator=g, device=dev) * 0.02 for r, c in _muon_shapes(case)]
        s['g'] = [_gradients(g, case['L'], r, c) for r, c in _muon_shapes(case)]
        s['m'] = [_gradients(g, case['L'], r, c) for r, c in _muon_shapes(case)]
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _whole(planes):
    return planes[0].float() + planes[1].float() if planes.shape[0] == 2 else planes[0].float()


def _planes_of(x, pair):
    hi = x.to(torch.bfloat16)
    return torch.stack([hi, (x - hi.float()).to(torch.bfloat16)]) if pair else hi[None]


def _angles(s):
    """cos / sin of every row [rows, 1, hd/2]"""
    case = s['case']
    rows, T = case['B'] * case['N'], case['N']
    if s['pos'] is None:
        i = torch.arange(rows, device=s['qkv'].device) % T
        return s['cos'][i][:, None], s['sin'][i][:, None]
    i = s['pos'].long()
    on = ((i >= 0) & (i < T))[:, None]
    i = i.clamp(0, T - 1)
    return torch.where(on, s['cos'][i], 1.0)[:, None], torch.where(on, s['sin'][i], 0.0)[:, None]


def _halves(z, inter):
    return (z[..., 0::2], z[..., 1::2]) if inter else z.chunk(2, -1)


def _joined(a, b, inter):
    return torch.stack([a, b], -1).flatten(-2) if inter else torch.cat([a, b], -1)


def _heads(s, x):
    case = s['case']
    x = x.view(x.shape[0], case['H'] + 2 * case['Hkv'], case['hd'])
    return x[:, :case['H']], x[:, case['H']:case['H'] + case['Hkv']], x[:, case['H'] + case['Hkv']:]


def _qk_plain(s):
    case, inter = s['case'], s['case']['inter']
    cos, sin = _angles(s)

    def one(x, gain):
        z = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        if gain is not None:
            z = z * gain
        a, b = _halves(z, inter)
        return _joined(a * cos - b * sin, b * cos + a * sin, inter)
    q, k, v = _heads(s, _whole(s['qkv']))
    out = torch.cat([one(q, s['gq']), one(k, s['gk']), v], 1).flatten(1)
    return _planes_of(out, case['pair'])


def _qk_plain_back(s):
    case, inter = s['case'], s['case']['inter']
    cos, sin = _angles(s)

    def one(dy, x, gain):
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        xh = x * r
        a, b = _halves(dy, inter)
        dz = _joined(a * cos + b * sin, b * cos - a * sin, inter)
        dgain = (dz * xh).sum((0, 1))
        d = dz * gain if gain is not None else dz
        return r * (d - xh * (d * xh).mean(-1, keepdim=True)), dgain
    q, k, _ = _heads(s, _whole(s['qkv']))
    dq, dk, dv = _heads(s, _whole(s['dout']))
    dq, dgq = one(dq, q, s['gq'])
    dk, dgk = one(dk, k, s['gk'])
    return _planes_of(torch.cat([dq, dk, dv], 1).flatten(1), case['pair']), dgq, dgk


def _ortho_plain(x, exact32):
    """x [L, r, c], any float type; 32 bits, or 64 where the result keeps 32: five steps multiply a rounding by up to 3.4^5"""
    x = x.double() if exact32 else x.float()
    tall = x.shape[1] > x.shape[2]
    x = x.mT.contiguous() if tall else x
    x = x / torch.sqrt((x * x).sum((1, 2), keepdim=True)).clamp(min=NORM_EPS)
    for _ in range(STEPS):
        A = torch.bmm(x, x.mT.contiguous())
        x = COEFF[0] * x + torch.bmm(COEFF[1] * A + COEFF[2] * torch.bmm(A, A), x)
    return x.mT if tall else x


def _muon_plain(s):
    lr, mu, wd, gs = s['hyper']
    for p, g, m in zip(s['p'], s['g'], s['m']):
        g = g * gs
        m.copy_(m * mu + g * (1 - mu))
        u = g * (1 - mu) + m * mu if s['case']['nesterov'] else m
        o = _ortho_plain(u, False)
        p.copy_(p * (1 - lr * wd) - lr * (0.2 * math.sqrt(max(p.shape[1:]))) * o)
    return s['p'], s['m']


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s['case']
    if case['op'] == 'qk':
        if own:
            from simple3d_former_amd import ops
            lo = lambda t: t[1] if case['pair'] else None  # noqa: E731
            kw = dict(Hkv=case['Hkv'], q_gain=s['gq'], k_gain=s['gk'], rope=(s['cos'], s['sin']), pos=s['pos'], eps=EPS, interleaved=case['inter'])
            out = torch.empty_like(s['qkv'])
            if case['back']:
                _, _, dgq, dgk = ops.qk_norm_rope_bwd(s['dout'][0], lo(s['dout']), s['qkv'][0], lo(s['qkv']), case['H'], case['hd'],
                                                      out=(out[0], lo(out)), **kw)
            else:
                ops.qk_norm_rope_fwd(s['qkv'][0], lo(s['qkv']), case['H'], case['hd'], out=(out[0], lo(out)), **kw)
        elif case['back']:
            out, dgq, dgk = _qk_plain_back(s)
        else:
            out = _qk_plain(s)
        # a pair of planes stands for its sum
        out = out.sum(0, dtype=torch.float32) if case['pair'] else out[0]
        return dict(dqkv=out, dgq=dgq, dgk=dgk) if case['back'] else dict(qkv=out)
    if case['op'] == 'ortho':
        dst = getattr(torch, case['dst'])
        if own:
            from simple3d_former_amd import ops
            return ops.orthogonalize(s['x'], steps=STEPS, coefficients=COEFF, eps=NORM_EPS, out_dtype=dst)
        return _ortho_plain(s['x'], case['dst'] == 'float32').to(dst)
    if own:
        from simple3d_former_amd import ops
        ops.muon_step(s['p'], s['g'], s['m'], s['hyper'], nesterov=case['nesterov'], steps=STEPS, coefficients=COEFF, eps=NORM_EPS,
                      scale='match_rms_adamw')
        p, m = s['p'], s['m']
    else:
        p, m = _muon_plain(s)
    return dict(p=p, m=m)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _ortho_exact(x):
    """The iteration written in A: every X is Q(A0) X0 with Q a product of commuting matrices, A <- P A P."""
    x = x.double()
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2).contiguous() if tall else x
    x = x / x.flatten(1).norm(dim=1).clamp(min=NORM_EPS)[:, None, None]
    A = torch.bmm(x, x.transpose(1, 2).contiguous())
    eye = torch.eye(A.shape[1], dtype=A.dtype, device=A.device)
    Q = eye.expand_as(A).contiguous()
    for _ in range(STEPS):
        P = COEFF[0] * eye + torch.bmm(A, COEFF[1] * eye + COEFF[2] * A)
        Q = torch.bmm(P, Q)
        A = torch.bmm(torch.bmm(P, A), P)
    x = torch.bmm(Q, x)
    return x.transpose(1, 2) if tall else x


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'ortho':
        return _ortho_exact(s['x'])
    if case['op'] == 'muon':
        lr, mu, wd, gs = s['hyper'].double()
        ps, ms = [], []
        for p, g, m in zip(s['p'], s['g'], s['m']):
            p, g, m = p.double(), g.double() * gs, m.double()
            m = m + (1 - mu) * (g - m)
            u = g + mu * (m - g) if case['nesterov'] else m
            ps.append(p - lr * (wd * p + 0.2 * max(p.shape[1:]) ** 0.5 * _ortho_exact(u)))
            ms.append(m)
        return dict(p=ps, m=ms)
    # qk: a pair of features is one complex number, the position's rotation its product with exp(i angle); the backward is autograd's
    H, Hkv, hd, N = case['H'], case['Hkv'], case['hd'], case['N']
    x = s['qkv'].double().sum(0).view(-1, H + 2 * Hkv, hd)
    rows = x.shape[0]
    turn = torch.complex(s['cos'].double(), s['sin'].double())
    turn = torch.cat([turn, torch.ones_like(turn[:1])])
    at = torch.arange(rows, device=x.device) % N if s['pos'] is None else torch.where((s['pos'] >= 0) & (s['pos'] < N), s['pos'], N).long()
    ones = torch.ones(hd, dtype=torch.float64, device=x.device)
    gq, gk = (ones if t is None else t.double() for t in (s['gq'], s['gk']))
    leaves = [t.requires_grad_(case['back']) for t in (x.contiguous(), gq.clone(), gk.clone())]

    def one(t, gain):
        t = t * gain / torch.sqrt(t.square().sum(-1, keepdim=True) / hd + EPS)
        t = t.unflatten(-1, (hd // 2, 2)) if case['inter'] else t.unflatten(-1, (2, hd // 2)).transpose(-1, -2)
        t = torch.view_as_real(torch.view_as_complex(t.contiguous()) * turn[at][:, None])
        return (t if case['inter'] else t.transpose(-1, -2)).flatten(-2)
    x, gq, gk = leaves
    y = torch.cat([one(x[:, :H], gq), one(x[:, H:H + Hkv], gk), x[:, H + Hkv:]], 1)
    if not case['back']:
        return dict(qkv=y.flatten(1))
    dx, dgq, dgk = torch.autograd.grad(y, leaves, s['dout'].double().sum(0).view_as(y))
    return dict(dqkv=dx.flatten(1), dgq=dgq, dgk=dgk)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _ortho_flops(L, r, c):
    m, n = min(r, c), max(r, c)
    return L * STEPS * (m * m * n + m * m * m + 2 * m * m * n)       # the two symmetric products need one half


def work(case):
    if case['op'] == 'qk':
        e = case['B'] * case['N'] * (case['H'] + 2 * case['Hkv']) * case['hd']
        e2 = 2 * e * (2 if case['pair'] else 1)
        table = case['N'] * case['hd'] * 4 + (4 * case['B'] * case['N'] if case['pos'] else 0)
        return dict(bytes=e2 * (3 if case['back'] else 2) + table, flops=e * (20 if case['back'] else 8))
    if case['op'] == 'ortho':
        size = dict(float32=4, bfloat16=2)
        e = case['L'] * case['r'] * case['c']
        return dict(bytes=e * (size[case['src']] + size[case['dst']]), flops=_ortho_flops(case['L'], case['r'], case['c']))
    e = sum(case['L'] * r * c for r, c in _muon_shapes(case))
    return dict(bytes=e * 20, flops=sum(_ortho_flops(case['L'], r, c) for r, c in _muon_shapes(case)))
