"""Thin tensor-level wrappers over the C ABI (one call = one libs3d_hip.so entry point).  Used by the parity tests and
by host code that needs a single operator; the training engine calls the same entry points directly."""
import ctypes

import torch

from . import _lib as L

EPI = dict(BF16_BIAS=0, GELU=1, RESID=2, TOKEN=3, F32=4, DGELU=5, ATOMIC=6, RELU=7, DRELU=8)


def _dev(t):
    assert t.is_cuda and t.is_contiguous(), 'device-resident contiguous tensor required'
    return t


def split_bf16(x, ld_out=None):
    """fp32 [rows, cols] -> (hi, lo) bf16 planes with x ~= hi + lo."""
    x = _dev(x.float())
    x2 = x.reshape(-1, x.shape[-1]) if x.dim() > 1 else x.reshape(1, -1)
    rows, cols = x2.shape
    ld = ld_out or cols
    hi = torch.zeros(rows, ld, dtype=torch.bfloat16, device=x.device)
    lo = torch.zeros_like(hi)
    L.check(L.lib().s3d_split_bf16(L.ptr(x2), L.ptr(hi), L.ptr(lo), ctypes.c_long(rows), ctypes.c_long(cols),
                                   ctypes.c_long(ld), L.current_stream()), 'split_bf16')
    return hi, lo


def gemm(ta, tb, split, epi, splitk=1, **fields):
    g = L.fill(L.S3dGemmArgs(), **fields)
    if 'alpha' not in fields:
        g.alpha = 1.0
    L.check(L.lib().s3d_gemm(int(ta), int(tb), int(split), EPI[epi] if isinstance(epi, str) else epi,
                             ctypes.byref(g), splitk, L.current_stream()), 'gemm')


def linear(x, w, bias=None, split=True):
    """y = x @ w^T + bias in fp32 out (x [M,K] fp32, w [N,K] fp32), via the (split-)bf16 MFMA GEMM."""
    M, K = x.shape
    N = w.shape[0]
    xh, xl = split_bf16(x)
    wh, wl = split_bf16(w)
    out = torch.empty(M, N, dtype=torch.float32, device=x.device)
    gemm(0, 0, split, 'F32', A_hi=xh, A_lo=xl, lda=K, B_hi=wh, B_lo=wl, ldb=K, M=M, N=N, K=K,
         bias=None if bias is None else _dev(bias.float()), C=out, ldc=N)
    return out


def layernorm_fwd(x, gamma, beta, eps=1e-6, want_f32=True):
    rows, D = x.shape
    hi = torch.empty(rows, D, dtype=torch.bfloat16, device=x.device)
    lo = torch.empty_like(hi)
    out = torch.empty(rows, D, dtype=torch.float32, device=x.device) if want_f32 else None
    mean = torch.empty(rows, dtype=torch.float32, device=x.device)
    rstd = torch.empty_like(mean)
    a = L.fill(L.S3dLnArgs(), x=_dev(x), ldx=D, rows=rows, D=D, eps=eps, gamma=_dev(gamma), beta=_dev(beta), out_hi=hi,
               out_lo=lo, out_f32=out, ldo=D, mean=mean, rstd=rstd)
    L.check(L.lib().s3d_layernorm_fwd(ctypes.byref(a), L.current_stream()), 'layernorm_fwd')
    return out, hi, lo, mean, rstd


def layernorm_bwd(dy, x, mean, rstd, gamma, dres=None):
    rows, D = x.shape
    dx = torch.empty_like(x)
    dx_bf = torch.empty(rows, D, dtype=torch.bfloat16, device=x.device)
    dg = torch.zeros(D, dtype=torch.float32, device=x.device)
    db = torch.zeros_like(dg)
    a = L.fill(L.S3dLnBwdArgs(), dy=_dev(dy), lddy=D, x=_dev(x), ldx=D, mean=mean, rstd=rstd, gamma=_dev(gamma),
               dres=dres, lddres=D, dx=dx, lddx=D, dx_bf=dx_bf, lddxbf=D, dgamma=dg, dbeta=db, rows=rows, D=D)
    L.check(L.lib().s3d_layernorm_bwd(ctypes.byref(a), L.current_stream()), 'layernorm_bwd')
    return dx, dx_bf, dg, db


def _drop_fields(drop):
    """drop = (p, seed tensor [1] int64 on the device, site) -> S3dAttnArgs / S3dGemmArgs dropout fields"""
    if not drop:
        return {}
    p, seed, site = drop
    return dict(drop_seed=seed, drop_site=int(site), drop_thr=int(p * 4294967296.0), drop_scale=1.0 / (1.0 - p))


def attention_fwd(qkv_hi, qkv_lo, Bb, H, N, D, sb, st, split=True, seg=0, drop=None, drop_mask=None, p_single_plane=0):
    rows = qkv_hi.shape[0]
    out_hi = torch.zeros(rows, D, dtype=torch.bfloat16, device=qkv_hi.device)
    out_lo = torch.zeros_like(out_hi)
    lse = torch.zeros(Bb * H * N, dtype=torch.float32, device=qkv_hi.device)
    a = L.fill(L.S3dAttnArgs(), qkv_hi=_dev(qkv_hi), qkv_lo=_dev(qkv_lo), ld=3 * D, out_hi=out_hi, out_lo=out_lo, ldo=D,
               lse=lse, Bb=Bb, H=H, N=N, D=D, sb=sb, st=st, scale=float((D // H) ** -0.5), seg=seg, drop_mask=drop_mask, p_single_plane=p_single_plane,
               **_drop_fields(drop))
    L.check(L.lib().s3d_attention_fwd(ctypes.byref(a), 1 if split else 0, L.current_stream()), 'attention_fwd')
    return out_hi, out_lo, lse


def attention_bwd(qkv_hi, out_hi, out_lo, lse, dout, Bb, H, N, D, sb, st, seg=0, drop=None, drop_mask=None):
    rows = qkv_hi.shape[0]
    dqkv = torch.zeros(rows, 3 * D, dtype=torch.bfloat16, device=qkv_hi.device)
    delta = torch.zeros(Bb * H * N, dtype=torch.float32, device=qkv_hi.device)
    a = L.fill(L.S3dAttnArgs(), qkv_hi=_dev(qkv_hi), ld=3 * D, out_hi=_dev(out_hi), out_lo=out_lo, ldo=D, lse=lse, Bb=Bb,
               H=H, N=N, D=D, sb=sb, st=st, scale=float((D // H) ** -0.5), dout=_dev(dout), lddo=D, dqkv=dqkv,
               lddq=3 * D, delta=delta, seg=seg, drop_mask=drop_mask, **_drop_fields(drop))
    L.check(L.lib().s3d_attention_bwd(ctypes.byref(a), L.current_stream()), 'attention_bwd')
    return dqkv


def voxel_fold(x, cell, patch, mode, ntok_rows, kpad):
    B, _, V, _, _ = x.shape
    a = torch.zeros(2, ntok_rows, kpad, dtype=torch.bfloat16, device=x.device)
    fa = L.fill(L.S3dFoldArgs(), x=_dev(x), a_hi=a[0], a_lo=a[1], lda=kpad, B=B, V=V, c=cell, P=patch, mode=mode)
    L.check(L.lib().s3d_voxel_fold(ctypes.byref(fa), L.current_stream()), 'voxel_fold')
    return a


def cross_entropy(logits, target, weight=None, grad_scale=1.0):
    rows, C = logits.shape
    loss = torch.zeros(2, dtype=torch.float32, device=logits.device)
    dl = torch.empty_like(logits)
    a = L.fill(L.S3dCeArgs(), logits=_dev(logits), target=_dev(target), weight=weight, rows=rows, C=C, loss=loss,
               dlogits=dl, grad_scale=grad_scale)
    L.check(L.lib().s3d_cross_entropy(ctypes.byref(a), L.current_stream()), 'cross_entropy')
    return loss[0], dl


# ---------------------------------------------------------------------------------------------- head norm + position rotation
def _same_device(who, *tensors):
    """All tensors on the CURRENT device: the call is enqueued on the current stream of it.  (This and the checks below run before every launch of
    calls that last a few microseconds: one attribute of a tensor costs 0.1.)"""
    on = {t.get_device() for t in tensors if t is not None}
    if on and (min(on) < 0 or on != {torch.cuda.current_device()}):
        raise ValueError(f'{who}: every tensor must be on the current device, got {sorted({str(t.device) for t in tensors if t is not None})}')


def _plane(who, name, t, rows, width):
    """A [rows, width] bf16 plane with contiguous rows; returns its row pitch."""
    if t.dtype == torch.bfloat16 and t.shape == (rows, width):
        ld, unit = t.stride()
        if unit == 1:
            return ld if rows > 1 else max(ld, width)
    raise ValueError(f'{who}: {name} must be a bfloat16 [{rows}, {width}] tensor with contiguous rows, got {t.dtype} {tuple(t.shape)} {t.stride()}')


def _addr(t):
    return None if t is None else t.data_ptr()


def rope_table(coords, hd, base=10000.0):
    """cos / sin table [T, hd/2] (fp32) for s3d_qk_norm_rope: coords [T] positions or [T, A] coordinates on A axes (a voxel grid: A = 3).  Each
    axis gets (hd/2) // A pairs with angles x * base^(-j / pairs); pairs left over are not rotated.  Angles are formed in 64 bits, so
    that far positions keep their phase."""
    c = torch.as_tensor(coords)
    if c.dim() not in (1, 2) or hd % 16 or not 16 <= hd <= 256:
        raise ValueError(f'rope_table: coords [T] or [T, A] and a head dim that is a multiple of 16 up to 256, got {tuple(c.shape)}, {hd}')
    c = c.to(torch.float64)
    c = c[:, None] if c.dim() == 1 else c
    T, A = c.shape
    half, per = hd // 2, hd // 2 // max(A, 1)
    if A < 1 or per < 1:
        raise ValueError(f'rope_table: {A} axes for {half} pairs')
    freq = float(base) ** (-torch.arange(per, dtype=torch.float64, device=c.device) / per)
    ang = torch.zeros(T, half, dtype=torch.float64, device=c.device)
    ang[:, :A * per] = (c[:, :, None] * freq).reshape(T, A * per)
    return ang.cos().float(), ang.sin().float()


def _qk_args(who, qkv_hi, qkv_lo, H, hd, Hkv, q_gain, k_gain, rope, pos, st, eps, interleaved):
    """The checked argument block of either direction, rows, width and the planes' row pitch."""
    Hkv = H if Hkv is None else Hkv
    if qkv_hi.dim() != 2:
        raise ValueError(f'{who}: qkv must be [rows, (H + 2 Hkv) hd], got {tuple(qkv_hi.shape)}')
    rows, W = qkv_hi.shape[0], (H + 2 * Hkv) * hd
    ld = _plane(who, 'qkv_hi', qkv_hi, rows, W)
    if qkv_lo is not None and _plane(who, 'qkv_lo', qkv_lo, rows, W) != ld:
        raise ValueError(f'{who}: the planes of a pair need the same row pitch')
    for g in (q_gain, k_gain):
        if g is not None and (g.dtype != torch.float32 or g.shape != (hd,) or not g.is_contiguous()):
            raise ValueError(f'{who}: q_gain and k_gain must be contiguous float32 [{hd}] tensors')
    cos, sin = rope if rope is not None else (None, None)
    T = 0
    if cos is not None:
        T = cos.shape[0]
        for t in (cos, sin):
            if t.dtype != torch.float32 or t.shape != (T, hd // 2) or not t.is_contiguous():
                raise ValueError(f'{who}: the rotation tables must be contiguous float32 [T, {hd // 2}] tensors')
    if pos is not None and (pos.dtype != torch.int32 or pos.shape != (rows,) or not pos.is_contiguous()):
        raise ValueError(f'{who}: pos must be a contiguous int32 [{rows}] tensor')
    a = L.S3dQkNormArgs(qkv_hi=qkv_hi.data_ptr(), qkv_lo=_addr(qkv_lo), ld=ld, rows=rows, H=H, Hkv=Hkv, hd=hd, eps=eps, q_gain=_addr(q_gain),
                        k_gain=_addr(k_gain), cos_t=_addr(cos), sin_t=_addr(sin), T=T, st=st, pos=_addr(pos), interleaved=1 if interleaved else 0)
    return a, rows, W


def _pair_out(who, name, out, like_hi, like_lo, rows, W):
    if out is None:
        return like_hi.new_empty((rows, W)), None if like_lo is None else like_hi.new_empty((rows, W)), W
    hi, lo = out
    ld = _plane(who, name, hi, rows, W)
    if lo is not None and _plane(who, name + ' (low plane)', lo, rows, W) != ld:
        raise ValueError(f'{who}: the planes of a pair need the same row pitch')
    return hi, lo, ld


def qk_norm_rope_fwd(qkv_hi, qkv_lo, H, hd, *, Hkv=None, q_gain=None, k_gain=None, rope=None, pos=None, st=1, eps=1e-6, interleaved=False, out=None):
    """Root-mean-square norm of every query / key head (gains [hd] fp32, None = 1) and rotation by the token's position, values copied:
    s3d_qk_norm_rope_fwd.  qkv planes [rows, (H + 2 Hkv) hd] bf16 (qkv_lo None: plain bf16); rope = (cos, sin) of rope_table or None;
    pos [rows] int32 table rows (outside the table: not rotated) or None: row r takes (r // st) % T.  out = (hi, lo) to write into, which may
    be the input planes; -> (out_hi, out_lo)."""
    who = 'qk_norm_rope_fwd'
    _same_device(who, qkv_hi, qkv_lo, q_gain, k_gain, pos, *(rope or ()), *(out or ()))
    a, rows, W = _qk_args(who, qkv_hi, qkv_lo, H, hd, Hkv, q_gain, k_gain, rope, pos, st, eps, interleaved)
    hi, lo, a.ldo = _pair_out(who, 'out', out, qkv_hi, qkv_lo, rows, W)
    if rows:
        a.out_hi, a.out_lo = hi.data_ptr(), _addr(lo)
        L.check(L.lib().s3d_qk_norm_rope_fwd(ctypes.byref(a), L.current_stream()), who)
    return hi, lo


def qk_norm_rope_bwd(dout_hi, dout_lo, qkv_hi, qkv_lo, H, hd, *, Hkv=None, q_gain=None, k_gain=None, rope=None, pos=None, st=1, eps=1e-6,
                     interleaved=False, out=None, gain_grads=None):
    """Backward of qk_norm_rope_fwd: dout planes (gradient of its output) and the INPUT qkv planes of the forward -> (dqkv_hi, dqkv_lo, dq_gain,
    dk_gain).  out = (hi, lo) to write dqkv into (may be the dout planes); gain_grads = (dq, dk) to ADD the gains' gradients to."""
    who = 'qk_norm_rope_bwd'
    _same_device(who, qkv_hi, qkv_lo, dout_hi, dout_lo, q_gain, k_gain, pos, *(rope or ()), *(out or ()), *(gain_grads or ()))
    a, rows, W = _qk_args(who, qkv_hi, qkv_lo, H, hd, Hkv, q_gain, k_gain, rope, pos, st, eps, interleaved)
    a.lddo = _plane(who, 'dout_hi', dout_hi, rows, W)
    if dout_lo is not None and _plane(who, 'dout_lo', dout_lo, rows, W) != a.lddo:
        raise ValueError(f'{who}: the planes of a pair need the same row pitch')
    hi, lo, a.lddq = _pair_out(who, 'out', out, dout_hi, dout_lo, rows, W)
    if gain_grads is None:
        dq, dk = (torch.empty(hd, dtype=torch.float32, device=qkv_hi.device) for _ in range(2))
    else:
        dq, dk = gain_grads
        for g in (dq, dk):
            if g.dtype != torch.float32 or g.shape != (hd,) or not g.is_contiguous():
                raise ValueError(f'{who}: the gains\' gradients must be contiguous float32 [{hd}] tensors')
    if rows:
        lib = L.lib()
        a.partial_blocks = lib.s3d_qk_norm_blocks(rows, a.H, a.Hkv, hd)
        part = torch.empty(a.partial_blocks * 2 * hd, dtype=torch.float32, device=qkv_hi.device)
        a.dout, a.dout_lo, a.dqkv, a.dqkv_lo = dout_hi.data_ptr(), _addr(dout_lo), hi.data_ptr(), _addr(lo)
        a.dq_gain, a.dk_gain, a.accumulate, a.partial = dq.data_ptr(), dk.data_ptr(), int(gain_grads is not None), part.data_ptr()
        L.check(lib.s3d_qk_norm_rope_bwd(ctypes.byref(a), L.current_stream()), who)
    elif gain_grads is None:
        dq.zero_()
        dk.zero_()
    return hi, lo, dq, dk


# ---------------------------------------------------------------------------------------------- orthogonalised updates
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _matrices(who, name, t, dtypes):
    """[r, c] or [L, r, c] with contiguous rows -> (count, rows, cols, stride, pitch)"""
    if t.dim() not in (2, 3) or t.dtype not in dtypes:
        raise ValueError(f'{who}: {name} must be a [rows, cols] or [count, rows, cols] tensor of {" / ".join(str(d) for d in dtypes)}, got {t.dtype} {tuple(t.shape)}')
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f'{who}: the rows of {name} must be contiguous')
    n = t.shape[0] if t.dim() == 3 else 1
    r, c = t.shape[-2:]
    ld = t.stride(-2) if r > 1 else max(c, 1)
    return n, r, c, (t.stride(0) if n > 1 else r * ld) if t.dim() == 3 else r * ld, ld


def _ns_args(steps, coefficients, eps, **kw):
    a, b, c = coefficients
    return L.S3dNsArgs(steps=steps, a=a, b=b, c=c, eps=eps, **kw)


def orthogonalize(x, *, steps=5, coefficients=NS_COEFFICIENTS, eps=1e-7, out_dtype=None, out=None):
    """Newton-Schulz orthogonalisation of a matrix [r, c] or a stack [L, r, c] (fp32 or bf16): s3d_orthogonalize.  The singular values of
    x / max(|x|_F, eps) go `steps` times through a s + b s^3 + c s^5, the singular vectors stay.  out_dtype: float32 or bfloat16 (the fp32
    result rounded once; default: x's); out: tensor to write into (may be x)."""
    who = 'orthogonalize'
    types = (torch.float32, torch.bfloat16)
    _same_device(who, x, out)
    n, r, c, xs, xld = _matrices(who, 'x', x, types)
    if out is None:
        out = torch.empty(x.shape, dtype=out_dtype or x.dtype, device=x.device)
    elif out.shape != x.shape or (out_dtype is not None and out.dtype != out_dtype):
        raise ValueError(f'{who}: out must have the shape of x and the requested type')
    _, _, _, os_, old = _matrices(who, 'out', out, types)
    it = L.S3dOrthoItem(x=x.data_ptr(), x_stride=xs, x_ld=xld, out=out.data_ptr(), out_stride=os_, out_ld=old, count=n, rows=r, cols=c)
    a = _ns_args(steps, coefficients, eps, x_bf16=int(x.dtype == torch.bfloat16), out_bf16=int(out.dtype == torch.bfloat16))
    lib = L.lib()
    size = lib.s3d_orthogonalize_workspace_bytes(ctypes.byref(it), 1, ctypes.byref(a))
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device=x.device)
    L.check(lib.s3d_orthogonalize(ctypes.byref(it), 1, ctypes.byref(a), ws.data_ptr(), size, L.current_stream()), who)
    return out


def muon_scale(scale, rows, cols):
    """Factor on the learning rate of a rows x cols update: 'original' sqrt(max(1, rows / cols)); 'match_rms_adamw' 0.2 sqrt(max(rows, cols)) (an
    update of the root mean square that Adam's has); or a number."""
    if scale == 'original':
        return max(1.0, rows / cols) ** 0.5
    if scale == 'match_rms_adamw':
        return 0.2 * max(rows, cols) ** 0.5
    return float(scale)


def muon_step(params, grads, momenta, hyper, *, planes=None, nesterov=True, steps=5, coefficients=NS_COEFFICIENTS, eps=1e-7, scale='original',
              zero_grad=False):
    """One optimizer step with orthogonalised momentum over matrix parameters, in place: s3d_muon_step.  params / grads / momenta: lists of fp32
    [r, c] or [L, r, c] tensors (one entry = one stack of equal matrices); hyper: fp32 device tensor {lr, momentum, decay, grad_scale};
    planes: list of (hi, lo) bf16 tensors laid out like the parameters, refreshed, or None.  scale: muon_scale's rule; VoxelEngine.set_muon
    chooses 'match_rms_adamw', whose updates are 0.2 sqrt(max(rows, cols)) times larger than plain ones ('original' on wide or square matrices)."""
    who = 'muon_step'
    f32 = (torch.float32,)
    if not len(params) == len(grads) == len(momenta) or (planes is not None and len(planes) != len(params)):
        raise ValueError(f'{who}: params, grads, momenta (and planes) must have the same length')
    _same_device(who, hyper, *params, *grads, *momenta, *[t for hl in planes or () for t in hl])
    if hyper.dtype != torch.float32 or hyper.numel() != 4 or not hyper.is_contiguous():
        raise ValueError(f'{who}: hyper must be a contiguous float32 tensor of 4 values')
    items = (L.S3dMuonItem * max(len(params), 1))()
    for i, (p, g, m) in enumerate(zip(params, grads, momenta)):
        if p.shape != g.shape or p.shape != m.shape:
            raise ValueError(f'{who}: parameter {i} {tuple(p.shape)}, its gradient {tuple(g.shape)} and momentum {tuple(m.shape)} differ')
        n, r, c, ps, pld = _matrices(who, f'params[{i}]', p, f32)
        _, _, _, gs, gld = _matrices(who, f'grads[{i}]', g, f32)
        _, _, _, ms, mld = _matrices(who, f'momenta[{i}]', m, f32)
        hi = lo = None
        if planes is not None:
            hi, lo = planes[i]
            for t in (hi, lo):
                if t.shape != p.shape or _matrices(who, f'planes[{i}]', t, (torch.bfloat16,))[3:] != (ps, pld):
                    raise ValueError(f'{who}: the planes of parameter {i} must be laid out like it')
        items[i] = L.S3dMuonItem(p=p.data_ptr(), p_stride=ps, p_ld=pld, g=g.data_ptr(), g_stride=gs, g_ld=gld, m=m.data_ptr(), m_stride=ms, m_ld=mld,
                                 hi=_addr(hi), lo=_addr(lo), count=n, rows=r, cols=c, scale=muon_scale(scale, r, c) if r and c else 0.0)
    a = _ns_args(steps, coefficients, eps, nesterov=int(bool(nesterov)), zero_grad=int(bool(zero_grad)))
    lib = L.lib()
    size = lib.s3d_muon_workspace_bytes(items, len(params), ctypes.byref(a))
    workspace = torch.empty(max(size, 16), dtype=torch.uint8, device=hyper.device)
    L.check(lib.s3d_muon_step(items, len(params), ctypes.byref(a), hyper.data_ptr(), workspace.data_ptr(), size, L.current_stream()), who)
