"""GPU: the state space block's operators (ops.causal_conv, ssm_scan, block_norm, GradNormClip and their gradients) against plain 64-bit
implementations.  Tolerances: `u` is half a step of the output's type (2^-24 f32, 2^-9 relative to the binade's top, i.e. 2^-8 of the value, bf16);
a result that is the sum of m terms computed in f32 is off by at most m * u32 * (the sum of the terms' absolute values) plus one rounding of
the output, and each v_exp_f32 / v_rcp_f32 / v_rsq_f32 adds a few u32 of the term that it is in."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def _dev():
    assert torch.cuda.is_available(), 'these tests need the MI355X'
    return torch.device('cuda:0')


def _rand(g, *shape):
    return torch.randn(shape, generator=g, dtype=torch.float64)


def _close(got, want, size, terms, what):
    """|got - want| <= half a step of got's type at `want` + terms * 2^-24 * size, elementwise; size = the sum of the terms' magnitudes."""
    got64, want = got.detach().cpu().double(), want.double()
    assert got64.shape == want.shape, (what, got64.shape, want.shape)
    tol = HALF[got.dtype] * want.abs() + terms * U32 * size + 1e-37
    bad = ~((got64 - want).abs() <= tol)
    assert not bad.any(), '%s: %d of %d off, worst %.3e against %.3e' % (
        what, int(bad.sum()), bad.numel(), float(((got64 - want).abs() - tol).max()), float(tol[bad].min()))


def _packed(lens, gap=0):
    """seq_off, seq_len (device) and the number of rows; `gap` rows of no sequence in front of each sequence and behind the last."""
    off, at = [], gap
    for m in lens:
        off.append(at)
        at += m + gap
    dev = _dev()
    return torch.tensor(off, dtype=torch.int64, device=dev), torch.tensor(lens, dtype=torch.int32, device=dev), at, off


# ------------------------------------------------------------------------------------------------------------- causal convolution


def _conv64(x, w, b, off, lens, state, silu, dy=None, dstate_out=None):
    """The definition per sequence, with autograd in f64; also the same with every term's magnitude (for the tolerances)."""
    K, D = w.shape[1], w.shape[0]
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b if b is not None else torch.zeros(D, dtype=torch.float64), state)]
    x, w, b, state = leaves
    y = torch.zeros_like(x)
    ys, last, obj = [], [], 0.0
    for s, (o, m) in enumerate(zip(off, lens)):
        ext = torch.cat([state[s], x[o:o + m]])
        v = sum(w[:, k] * ext[k:k + m] for k in range(K)) + b
        v = v * torch.sigmoid(v) if silu else v
        ys.append(v)
        last.append(ext[m:])
        if dy is not None:
            obj = obj + (v * dy[o:o + m]).sum() + ((ext[m:] * dstate_out[s]).sum() if dstate_out is not None else 0.0)
    grads = None if dy is None else torch.autograd.grad(obj, leaves)
    return [v.detach() for v in ys], torch.stack(last).detach(), grads


CONV = [  # lens, D, K, gap, pad (extra columns of the row tensors)
    ([1], 8, 2, 0, 0), ([0, 3, 1], 5, 4, 1, 3), ([16] * 7, 64, 4, 0, 0), ([257, 0, 2, 40], 132, 3, 2, 4), ([9, 8, 7, 33], 33, 8, 1, 0), ([65], 640, 4, 0, 8),
    ([5, 64, 31], 12, 6, 0, 4)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('silu', [True, False])
@pytest.mark.parametrize('lens,D,K,gap,pad', CONV)
def test_causal_conv_forward_and_backward(lens, D, K, gap, pad, silu, dtype):
    from dotaclient_amd import ops
    dev = _dev()
    g = torch.Generator().manual_seed(D * 100 + K)
    off_d, len_d, rows, off = _packed(lens, gap)
    n = len(lens)
    x, dy = _rand(g, rows, D + pad).to(dtype).to(dev), _rand(g, rows, D + pad).to(dtype).to(dev)
    w, b = (_rand(g, D, K) * K ** -0.5).float().to(dev), _rand(g, D).float().to(dev)
    state, dso = _rand(g, n, K - 1, D).to(dtype).to(dev), _rand(g, n, K - 1, D).to(dtype).to(dev)
    xv, dyv = x[:, pad:], dy[:, pad:]
    keep = torch.full((rows, D + pad), 7.0, dtype=dtype, device=dev)
    y, so = ops.causal_conv(xv, w, b, off_d, len_d, max(lens), state=state, silu=silu, y=keep[:, pad:])
    c = lambda t: t.cpu().double()                                                     # noqa: E731
    want, last, grads = _conv64(c(xv), c(w), c(b), off, lens, c(state), silu, c(dyv), c(dso))
    size, _, gsize = _conv64(c(xv).abs(), c(w).abs(), c(b).abs(), off, lens, c(state).abs(), False, c(dyv).abs(), c(dso).abs())
    inside = torch.zeros(rows, dtype=torch.bool)
    for s, (o, m) in enumerate(zip(off, lens)):
        inside[o:o + m] = True
        _close(y[o:o + m], want[s], 2 * size[s], 2 * K + 8, 'y of sequence %d' % s)
    assert torch.equal(keep[~inside.to(dev)], torch.full_like(keep[~inside.to(dev)], 7.0)) and (pad == 0 or torch.all(keep[:, :pad] == 7.0))
    assert torch.equal(c(so), last)
    dx, dw, db, dst = ops.causal_conv_backward(dyv, xv, w, b, off_d, len_d, max(lens), state=state, silu=silu, dstate_out=dso)
    # |silu'| <= 1.1, its own error a few steps of 1 + |v| (times the term): the magnitudes of the plain gradient, with the pre-activation's on top
    mag = 2.0 * (1.0 + max(float(s.max()) if s.numel() else 0.0 for s in size))
    terms = 3 * K + 16
    _close(dx[inside.to(dev)], grads[0][inside], mag * gsize[0][inside], terms, 'dx')
    # a gradient of the parameters adds up to `rows` terms: 8 rows in a thread, 8 chunks, partial sums in order
    _close(dw, grads[1], mag * gsize[1], terms + 64 + rows // 64, 'dweight')
    _close(db, grads[2], mag * gsize[2], terms + 64 + rows // 64, 'dbias')
    _close(dst, grads[3], mag * gsize[3], terms, 'dstate')
    # the same without a state and a bias
    y0, so0 = ops.causal_conv(xv, w, None, off_d, len_d, max(lens), silu=silu)
    want0, last0, _ = _conv64(c(xv), c(w), None, off, lens, torch.zeros(n, K - 1, D, dtype=torch.float64), silu)
    for s, (o, m) in enumerate(zip(off, lens)):
        _close(y0[o:o + m], want0[s], 2 * size[s], 2 * K + 8, 'y without state, sequence %d' % s)
    assert torch.equal(c(so0), last0)
    _, _, db0, dst0 = ops.causal_conv_backward(dyv, xv, w, None, off_d, len_d, max(lens), silu=silu)
    assert db0 is None and dst0 is None


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_causal_conv_steps_equal_the_sequence_and_chunks_carry_the_state(dtype):
    from dotaclient_amd import ops
    dev = _dev()
    g = torch.Generator().manual_seed(5)
    n, T, D, K = 10, 21, 48, 4
    x = _rand(g, n * T, D).to(dtype).to(dev)
    w, b = _rand(g, D, K).float().to(dev), _rand(g, D).float().to(dev)
    off = torch.arange(n, device=dev) * T
    ln = torch.full((n,), T, dtype=torch.int32, device=dev)
    y, last = ops.causal_conv(x, w, b, off, ln, T)
    state = torch.zeros(n, K - 1, D, dtype=dtype, device=dev)
    for t in range(T):
        yt, state = ops.causal_conv_step(x.view(n, T, D)[:, t], state, w, b, state_out=state if t % 2 else None)
        assert torch.equal(yt, y.view(n, T, D)[:, t]), t
    assert torch.equal(state, last)
    # two chunks of one sequence, the second one starting from the first one's state
    cut = 9
    y1, s1 = ops.causal_conv(x, w, b, off, torch.full_like(ln, cut), cut)
    y2, s2 = ops.causal_conv(x, w, b, off + cut, ln - cut, T - cut, state=s1)
    assert torch.equal(y1.view(n, T, D)[:, :cut], y.view(n, T, D)[:, :cut]) and torch.equal(y2.view(n, T, D)[:, cut:], y.view(n, T, D)[:, cut:])
    assert torch.equal(s2, last)


def test_causal_conv_reads_nothing_outside_its_window():
    # an infinity or NaN touches the K rows that its taps reach and no other row, sequence or channel (also for the widths without own kernels)
    from dotaclient_amd import ops
    dev = _dev()
    for K in (2, 3, 4, 5, 7, 8):
        off_d, len_d, rows, off = _packed([30, 30], 0)
        x = torch.ones(rows, 8, device=dev)
        x[10, 3] = float('inf')
        w = torch.full((8, K), 0.1, device=dev)
        y, _ = ops.causal_conv(x, w, None, off_d, len_d, 30, silu=False)
        bad = ~torch.isfinite(y)
        want = torch.zeros_like(bad)
        want[10:10 + K, 3] = True
        assert torch.equal(bad, want), K
        dx, dw, _, _ = ops.causal_conv_backward(x, torch.ones_like(x), w, None, off_d, len_d, 30, silu=False)
        want = torch.zeros_like(bad)
        want[10 - K + 1:11, 3] = True
        assert torch.equal(~torch.isfinite(dx), want), K


def test_causal_conv_sequences_that_point_outside_are_cut():
    from dotaclient_amd import ops
    dev = _dev()
    x = torch.randn(40, 16, device=dev)
    w = torch.randn(16, 3, device=dev)
    off = torch.tensor([0, 30, 41, -5, 1 << 40], dtype=torch.int64, device=dev)
    ln = torch.tensor([20, 4000, 7, 7, 9], dtype=torch.int32, device=dev)
    keep = torch.full_like(x, 3.0)
    y, _ = ops.causal_conv(x, w, None, off, ln, 16, y=keep)
    good, _ = ops.causal_conv(x, w, None, off[:2].contiguous(), torch.tensor([16, 10], dtype=torch.int32, device=dev), 16, y=torch.full_like(x, 3.0))
    assert torch.equal(y, good) and torch.all(y[16:30] == 3.0)


# ------------------------------------------------------------------------------------------------------------------- block norms


def _norm64(y, r, wp, z, s, wq, eps):
    g = y if z is None else y * z * torch.sigmoid(z)
    u = g / torch.sqrt((g * g).mean(-1, keepdim=True) + eps)
    r = r + (wp * u if s is None else s * wp * u)
    return r, None if wq is None else wq * r / torch.sqrt((r * r).mean(-1, keepdim=True) + eps)


@pytest.mark.parametrize('types', [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize('rows,D,parts,pad', [(1, 1, 'zsw', 0), (5, 16, 'zsw', 0), (130, 512, 'zsw', 4), (67, 513, '', 0), (33, 1000, 'zw', 0), (9, 1028, 'sw', 4),
                                              (7, 4096, 'zsw', 0), (3, 8191, 'z', 1), (4500, 24, 'zsw', 0)])
def test_block_norm_forward_and_backward(rows, D, parts, pad, types):
    from dotaclient_amd import ops
    dev = _dev()
    ty, tr = types
    eps = 1e-5
    g = torch.Generator().manual_seed(rows * 10000 + D)
    c = lambda t: None if t is None else t.cpu().double()                              # noqa: E731
    row = lambda d: _rand(g, rows, D + pad).to(d).to(dev)[:, pad:]                     # noqa: E731
    y, r, dr = row(ty), row(tr), row(tr)
    z = row(ty) if 'z' in parts else None
    s = _rand(g, D).float().to(dev) if 's' in parts else None
    wp = (1 + 0.1 * _rand(g, D)).float().to(dev)
    wq = (1 + 0.1 * _rand(g, D)).float().to(dev) if 'w' in parts else None
    dx = row(ty) if wq is not None else None
    ro, xo = ops.block_norm(y, r, wp, gate=z, scale=s, w_pre=wq, eps=eps)
    leaves = [None if t is None else t.requires_grad_(True) for t in (c(y), c(r), c(wp), c(z), c(s), c(wq))]
    rw, xw = _norm64(*leaves, eps)
    # u is off by the gate's few steps, the mean's (log-depth sums: 16 terms in a lane, 6 levels, 8 waves) and rsqrt's: 40 steps of its size
    post = (rw - leaves[1]).detach().abs()
    _close(ro, rw.detach(), post + rw.detach().abs(), 48, 'r')
    if wq is not None:
        inv = xw.detach().abs() / (rw.detach().abs() + 1e-300)
        _close(xo, xw.detach(), xw.detach().abs() + inv * (post + rw.detach().abs()), 96, 'x')
    else:
        assert xo is None
    have = [t for t in leaves if t is not None]
    obj = (rw * c(dr)).sum() + (0.0 if dx is None else (xw * c(dx)).sum())
    grads = iter(torch.autograd.grad(obj, have))
    want = [None if t is None else next(grads) for t in leaves]
    dy, dres, dwp, dz, ds, dwq = ops.block_norm_backward(dr, dx, y, r, wp, gate=z, scale=s, w_pre=wq, eps=eps)
    # magnitudes of the terms behind each gradient, from the formulas with absolute values
    f = lambda t, o: o if t is None else c(t)                                          # noqa: E731
    zz = f(z, None)
    sg = 1.0 if zz is None else (zz * torch.sigmoid(zz)).abs()
    gg = c(y) if zz is None else c(y) * zz * torch.sigmoid(zz)
    i1 = 1 / torch.sqrt((gg * gg).mean(-1, keepdim=True) + eps)
    u = (gg * i1).abs()
    R = c(dr).abs()
    if wq is not None:
        i2 = 1 / torch.sqrt((rw.detach() ** 2).mean(-1, keepdim=True) + eps)
        v = (c(r).abs() + post) * i2
        e = (c(dx) * c(wq)).abs()
        R = R + i2 * (e + v * (e * v).mean(-1, keepdim=True))
    du = R * f(s, torch.ones(())).abs() * c(wp).abs()
    dg = i1 * (du + u * (du * u).mean(-1, keepdim=True))
    col = 200 + rows // 8
    _close(dres, want[1], R, 160, 'dresidual')
    _close(dy, want[0], dg * sg, 240, 'dy')
    _close(dwp, want[2], (R * f(s, torch.ones(())).abs() * u).sum(0), col, 'dw_post')
    if z is not None:
        _close(dz, want[3], dg * c(y).abs() * torch.sigmoid(zz) * (1 + zz.abs()), 240, 'dgate')
    if s is not None:
        _close(ds, want[4], (R * c(wp).abs() * u).sum(0), col, 'dscale')
    if wq is not None:
        _close(dwq, want[5], (c(dx).abs() * v).sum(0), col, 'dw_pre')
    assert (dz is None) == (z is None) and (ds is None) == (s is None) and (dwq is None) == (wq is None)
    # in place on the residual stream
    if pad == 0:
        r2 = r.clone()
        ro2, xo2 = ops.block_norm(y, r2, wp, gate=z, scale=s, w_pre=wq, eps=eps, residual_out=r2)
        assert ro2.data_ptr() == r2.data_ptr() and torch.equal(ro2, ro) and (xo is None or torch.equal(xo2, xo))


# -------------------------------------------------------------------------------------------------------------- gradient clipping


@pytest.mark.parametrize('sizes', [[1], [0, 7, 0, 16384, 16385, 3, 0], [229376, 896, 256, 154], [5] * 300, [100003, 1, 65536]])
@pytest.mark.parametrize('mixed', [False, True])
def test_grad_norm_clip(sizes, mixed):
    from dotaclient_amd import ops
    dev = _dev()
    g = torch.Generator().manual_seed(len(sizes) + sizes[-1])
    base = [_rand(g, n + 1).to(torch.bfloat16 if mixed and i % 2 else torch.float32).to(dev) for i, n in enumerate(sizes)]
    grads = [t[1:] if i % 3 == 2 else t[:-1] for i, t in enumerate(base)]              # some start off a 16-byte boundary
    before = [t.clone() for t in grads]
    norms64 = torch.stack([t.cpu().double().norm() for t in grads])
    total64 = norms64.norm()
    # sums in f64, one rounding of the norm; c rounds twice more, its product once
    for factor, inplace in ((0.25, False), (4.0, False), (0.25, True), (4.0, True)):
        out = None if inplace else [torch.full_like(t, 9.0) for t in grads]
        clip = ops.GradNormClip(grads, out)
        total, norms = clip(factor * float(total64))
        _close(total[None], total64[None], total64[None], 1, 'total')
        _close(norms, norms64, norms64, 1, 'norms')
        c = min(1.0, factor * float(total64) / (float(total64) + 1e-6))
        for i, (a, b) in enumerate(zip(grads if inplace else out, before)):
            _close(a, b.cpu().double() * c, b.cpu().double().abs(), 4, 'tensor %d' % i)
            if c == 1.0:
                assert torch.equal(a, b)
        for a, b in zip(grads, before):
            a.copy_(b)
    edge = [t[:1] if i % 3 == 2 else t[-1:] for i, t in enumerate(base)]
    assert all(torch.isfinite(t).all() for t in edge)


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_grad_norm_clip_of_a_norm_that_is_not_finite_changes_nothing(bad):
    from dotaclient_amd import ops
    dev = _dev()
    grads = [torch.randn(1000, device=dev), torch.randn(50, device=dev).bfloat16()]
    grads[1][3] = bad
    before = [t.clone() for t in grads]
    total, norms = ops.grad_norm_clip(grads, 0.5)
    assert not torch.isfinite(total) and torch.isfinite(norms[0]) and not torch.isfinite(norms[1])
    assert all(torch.equal(a.nan_to_num(1.5), b.nan_to_num(1.5)) for a, b in zip(grads, before))
    # and the largest finite values do not overflow on the way: squares are summed in f64
    big = [torch.full((1000,), 1e30, device=dev)]
    total, _ = ops.grad_norm_clip(big, 1.0)
    assert abs(float(total) / (1e30 * 1000 ** 0.5) - 1) < 1e-6 and torch.isfinite(big[0]).all() and float(big[0].norm()) < 1.001


def test_grad_norm_clip_follows_its_tensors():
    """A gradient that is given other memory, of another size too, after the handle was built is clipped where it is then; the old memory stays as it was."""
    from dotaclient_amd import ops
    dev = _dev()
    a, b = torch.full((1000,), 2.0, device=dev), torch.full((77,), 1.0, device=dev)
    old = a.data
    clip = ops.GradNormClip([a, b])
    clip(1e9)
    a.data = torch.full((5000,), 3.0, device=dev)
    total, norms = clip(1.0)
    want = (5000 * 9 + 77) ** 0.5
    assert abs(float(total) - want) < 1e-6 * want and abs(float(norms[0]) - 45000 ** 0.5) < 1e-6 * want
    assert torch.allclose(a, torch.full_like(a, 3 / want), rtol=1e-6) and torch.allclose(b, torch.full_like(b, 1 / want), rtol=1e-6)
    assert torch.equal(old, torch.full_like(old, 2.0))
    b.data = a.data[100:177]
    with pytest.raises(ValueError, match='overlap'):
        clip(1.0)


# ----------------------------------------------------------------------------------------------------------- state space scan


def _scan64(x, dt, la, B, C, D, h0, off, lens):
    """The recurrence in f64, row by row; la = log decays [rows, H], dt the step sizes (both after bias and softplus)."""
    rep = x.shape[1] // B.shape[1]
    ys, hs = [], []
    for s, (o, m) in enumerate(zip(off, lens)):
        h = h0[s]
        for t in range(o, o + m):
            Bt, Ct = B[t].repeat_interleave(rep, 0), C[t].repeat_interleave(rep, 0)
            h = h * torch.exp(la[t])[:, None, None] + (dt[t][:, None] * x[t])[:, :, None] * Bt[:, None]
            ys.append((h * Ct[:, None]).sum(-1) + D[:, None] * x[t])
        hs.append(h)
    return (torch.stack(ys) if ys else x[:0]), torch.stack(hs)


def _scan_reference(i, off, lens, softplus):
    """Values, gradients and the magnitudes of the sums behind them, all f64 on the CPU.  i: the inputs as f64 tensors."""
    raw = (i['dt'] + i['bias']).requires_grad_(True)
    leaves = {k: i[k].clone().requires_grad_(True) for k in ('x', 'A', 'B', 'C', 'D', 'h0')}
    d = torch.nn.functional.softplus(raw) if softplus else raw
    y, hT = _scan64(leaves['x'], d, d * leaves['A'], leaves['B'], leaves['C'], leaves['D'], leaves['h0'], off, lens)
    rows_in = torch.cat([torch.arange(o, o + m) for o, m in zip(off, lens)]) if sum(lens) else torch.zeros(0, dtype=torch.long)
    obj = (y * i['dy'][rows_in]).sum() + (hT * i['dhT']).sum()
    keys = ['raw'] + list(leaves)
    got = dict(zip(keys, torch.autograd.grad(obj, [raw] + list(leaves.values()))))
    # magnitudes: everything non-negative, the decays as they are
    ab = {k: i[k].abs().requires_grad_(True) for k in ('x', 'B', 'C', 'D', 'h0')}
    dm, la = d.detach().abs().requires_grad_(True), (d * i['A']).detach().requires_grad_(True)
    ya, ha = _scan64(ab['x'], dm, la, ab['B'], ab['C'], ab['D'], ab['h0'], off, lens)
    obja = (ya * i['dy'][rows_in].abs()).sum() + (ha * i['dhT'].abs()).sum()
    keys = ['d', 'la'] + list(ab)
    size = dict(zip(keys, torch.autograd.grad(obja, [dm, la] + list(ab.values()))))
    # the kernel's way to d(la): differences of sums over the rows behind, inside a block of 64
    flow = torch.zeros_like(size['la'])
    ydy = torch.zeros_like(flow)
    ydy[rows_in] = (ya.detach() * i['dy'][rows_in].abs()).sum(-1)
    xdx = (ab['x'].detach() * size['x']).sum(-1)
    for o, m in zip(off, lens):
        for t0 in range(0, m, 64):
            sl = slice(o + t0, o + min(m, t0 + 64))
            flow[sl] = (ydy[sl] + xdx[sl]).flip(0).cumsum(0).flip(0)
    size['la'] = size['la'] + flow
    slope = torch.sigmoid(raw.detach()) if softplus else torch.ones_like(raw.detach())
    inside = torch.zeros(raw.shape[0], 1, dtype=torch.float64)
    inside[rows_in] = 1.0
    size['raw'] = (size['d'] + size['la'] * i['A'].abs()) * slope
    size['A'] = (size['la'] * d.detach() * inside).sum(0)
    size['bias'] = size['raw'].sum(0)
    got['bias'] = got['raw'].sum(0)
    return dict(y=y.detach(), hT=hT.detach(), rows=rows_in, grads=got, size=size, ya=ya.detach(), ha=ha.detach())


def _scan_inputs(seed, lens, gap, H, P, G, N, dtype, pad):
    off_d, len_d, rows, off = _packed(lens, gap)
    g = torch.Generator().manual_seed(seed)
    dev, n = _dev(), len(lens)
    wide = _rand(g, rows, pad + H * P + 2 * G * N).to(dtype).to(dev)
    dev_in = dict(x=wide[:, pad:pad + H * P].unflatten(1, (H, P)), B=wide[:, pad + H * P:pad + H * P + G * N].unflatten(1, (G, N)),
                  C=wide[:, pad + H * P + G * N:].unflatten(1, (G, N)), dt=_rand(g, rows, H).to(dtype).to(dev),
                  A=-(1 + 15 * torch.rand(H, generator=g)).to(dev), D=_rand(g, H).float().to(dev),
                  bias=(torch.rand(H, generator=g) * 4 - 6).to(dev), h0=_rand(g, n, H, P, N).float().to(dev),
                  dy=_rand(g, rows, H, P).to(dtype).to(dev), dhT=_rand(g, n, H, P, N).float().to(dev))
    return off_d, len_d, rows, off, dev_in


SCAN = [  # lens, gap, H, P, G, N, pad
    ([1], 0, 1, 1, 1, 1, 0), ([2, 0, 3], 1, 2, 8, 1, 8, 0), ([64], 0, 1, 64, 1, 64, 0), ([65, 63, 0, 128], 2, 2, 64, 1, 32, 8), ([16] * 9, 0, 4, 32, 2, 16, 0),
    ([130, 7], 0, 3, 48, 3, 40, 8), ([71], 3, 2, 77, 1, 101, 1), ([200], 0, 2, 128, 1, 128, 0), ([33, 90], 0, 6, 40, 2, 24, 0), ([300], 0, 1, 64, 1, 128, 0),
    ([513], 0, 1, 17, 1, 33, 0)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('softplus', [True, False])
@pytest.mark.parametrize('lens,gap,H,P,G,N,pad', SCAN)
def test_ssm_scan_forward_and_backward(lens, gap, H, P, G, N, pad, softplus, dtype):
    from dotaclient_amd import ops
    dev = _dev()
    off_d, len_d, rows, off, d = _scan_inputs(sum(lens) * 31 + P * N, lens, gap, H, P, G, N, dtype, pad)
    if not softplus:                                       # step sizes as they are: small and positive
        d['dt'] = (d['dt'].float().abs() * 0.05).to(dtype)
        d['bias'] = d['bias'].abs() * 1e-3
    i64 = {k: v.cpu().double() for k, v in d.items()}
    ref = _scan_reference(i64, off, lens, softplus)
    keep = torch.full((rows, H, P), 7.0, dtype=dtype, device=dev)
    seqs = (off_d, len_d, max(lens))
    kw = dict(D=d['D'], dt_bias=d['bias'], h0=d['h0'], softplus=softplus)
    y, hT = ops.ssm_scan(d['x'], d['dt'], d['A'], d['B'], d['C'], *seqs, y=keep, **kw)
    inside = ref['rows'].to(dev)
    # f32: sums of up to 64 + N + P terms, a few steps per factor (exp of differences up to ~100: 100 of them), 16 per block and segment on the
    # way.  bf16: the factors G1 L dt and S are rounded once (half a step of the term) for y, dx, dB, dC; what ends in f32 is made of three
    # bf16 pieces per factor, exact to 2^-24.
    bf = dtype == torch.bfloat16
    terms = 64 + N + P + 160 + 32 * (1 + max(lens) // 64)
    f32_terms = terms + (8 if bf else 0)
    out_terms = terms + (2 ** 16 if bf else 0)             # 2^-8 of the sum of the terms' magnitudes
    _close(y[inside], ref['y'], ref['ya'], out_terms, 'y')
    rest = torch.ones(rows, dtype=torch.bool)
    rest[ref['rows']] = False
    assert torch.all(y[rest.to(dev)] == 7.0)
    _close(hT, ref['hT'], ref['ha'], f32_terms, 'hT')
    g = ops.ssm_scan_backward(d['dy'], d['x'], d['dt'], d['A'], d['B'], d['C'], *seqs, dhT=d['dhT'], **kw)
    G_, S_ = ref['grads'], ref['size']
    _close(g.dx[inside], G_['x'][ref['rows']], S_['x'][ref['rows']], out_terms, 'dx')
    _close(g.dB[inside], G_['B'][ref['rows']], S_['B'][ref['rows']], 2 * out_terms, 'dB')
    _close(g.dC[inside], G_['C'][ref['rows']], S_['C'][ref['rows']], 2 * out_terms, 'dC')
    _close(g.ddt[inside], G_['raw'][ref['rows']], S_['raw'][ref['rows']], 2 * f32_terms, 'ddt')
    _close(g.dA, G_['A'], S_['A'], 2 * f32_terms, 'dA')
    _close(g.dD, G_['D'], S_['D'], f32_terms, 'dD')
    _close(g.ddt_bias, G_['bias'], S_['bias'], 2 * f32_terms, 'ddt_bias')
    _close(g.dh0, G_['h0'], S_['h0'], f32_terms, 'dh0')


def test_ssm_scan_without_its_optional_inputs():
    from dotaclient_amd import ops
    dev = _dev()
    lens = [70, 5]
    off_d, len_d, rows, off, d = _scan_inputs(3, lens, 0, 2, 64, 1, 64, torch.float32, 0)
    d['dt'] = d['dt'].abs() * 0.05
    i64 = {k: v.cpu().double() for k, v in d.items()}
    for k in ('bias', 'D', 'h0', 'dhT'):
        i64[k] = torch.zeros_like(i64[k])
    ref = _scan_reference(i64, off, lens, False)
    y, hT = ops.ssm_scan(d['x'], d['dt'], d['A'], d['B'], d['C'], off_d, len_d, 70)
    _close(y, ref['y'], ref['ya'], 500, 'y')
    _close(hT, ref['hT'], ref['ha'], 500, 'hT')
    g = ops.ssm_scan_backward(d['dy'], d['x'], d['dt'], d['A'], d['B'], d['C'], off_d, len_d, 70)
    assert g.dD is None and g.ddt_bias is None and g.dh0 is None
    _close(g.dx, ref['grads']['x'], ref['size']['x'], 1000, 'dx')
    _close(g.ddt, ref['grads']['raw'], ref['size']['raw'], 1000, 'ddt')
    _close(g.dA, ref['grads']['A'], ref['size']['A'], 1000, 'dA')


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,H,G', [(1100, 2, 1), (530, 4, 2)])
def test_ssm_scan_many_short_sequences(n, H, G, dtype):
    # more sequences than the slot table takes in one go, enough blocks for a workgroup to take all heads of a group; offsets not in order
    from dotaclient_amd import ops
    dev = _dev()
    P, N = 16, 8
    lens = [1 + (7 * k) % 3 for k in range(n)]
    off_d, len_d, rows, off, d = _scan_inputs(n, lens, 0, H, P, G, N, dtype, 0)
    order = torch.randperm(n, generator=torch.Generator().manual_seed(1))
    off, lens = [off[k] for k in order], [lens[k] for k in order]
    off_d, len_d = off_d[order.to(dev)].contiguous(), len_d[order.to(dev)].contiguous()
    i64 = {k: v.cpu().double() for k, v in d.items()}
    ref = _scan_reference(i64, off, lens, True)
    kw = dict(D=d['D'], dt_bias=d['bias'], h0=d['h0'], softplus=True)
    y, hT = ops.ssm_scan(d['x'], d['dt'], d['A'], d['B'], d['C'], off_d, len_d, 3, **kw)
    r = ref['rows'].to(dev)
    out = 300 + (2 ** 16 if dtype == torch.bfloat16 else 0)
    _close(y[r], ref['y'], ref['ya'], out, 'y')
    _close(hT, ref['hT'], ref['ha'], 300, 'hT')
    g = ops.ssm_scan_backward(d['dy'], d['x'], d['dt'], d['A'], d['B'], d['C'], off_d, len_d, 3, dhT=d['dhT'], **kw)
    G_, S_ = ref['grads'], ref['size']
    for name, got, terms in (('x', g.dx, out), ('B', g.dB, 2 * out), ('C', g.dC, 2 * out), ('raw', g.ddt, 600)):
        _close(got[r], G_[name][ref['rows']], S_[name][ref['rows']], terms, name)
    for name, got in (('A', g.dA), ('D', g.dD), ('bias', g.ddt_bias), ('h0', g.dh0)):
        _close(got, G_[name], S_[name], 600, name)


def _outputs(ops, d, seqs, softplus=True):
    kw = dict(D=d['D'], dt_bias=d['bias'], h0=d['h0'], softplus=softplus)
    return list(ops.ssm_scan(d['x'], d['dt'], d['A'], d['B'], d['C'], *seqs, **kw)) + \
        list(ops.ssm_scan_backward(d['dy'], d['x'], d['dt'], d['A'], d['B'], d['C'], *seqs, dhT=d['dhT'], **kw))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_ssm_scan_reads_only_its_sequences_and_repeats_itself(dtype):
    # what lies between the sequences may be anything; the same call gives the same bits
    from dotaclient_amd import ops
    lens = [70, 0, 1, 129, 5]
    off_d, len_d, rows, off, d = _scan_inputs(11, lens, 3, 4, 64, 2, 64, dtype, 8)
    seqs = (off_d, len_d, 200)                             # max_len may be more than the longest
    first = _outputs(ops, d, seqs)
    again = _outputs(ops, d, seqs)
    gaps = torch.ones(rows, dtype=torch.bool, device=_dev())
    for o, m in zip(off, lens):
        gaps[o:o + m] = False
    for k in ('x', 'B', 'C', 'dt', 'dy'):
        d[k][gaps] = float('nan')
    spoiled = _outputs(ops, d, seqs)
    for k, (a, b, c) in enumerate(zip(first, again, spoiled)):
        if a.shape[0] == rows:
            a, b, c = a[~gaps], b[~gaps], c[~gaps]
        assert torch.isfinite(a).all(), k
        assert torch.equal(a, b) and torch.equal(a, c), k


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_ssm_scan_extreme_step_sizes(dtype):
    # decays that underflow to nothing, and none at all
    from dotaclient_amd import ops
    off_d, len_d, rows, off, d = _scan_inputs(12, [150], 0, 2, 16, 1, 16, dtype, 0)
    d['A'] = torch.tensor([-1.0, -16.0], device=_dev())
    dt = torch.zeros(rows, 2)
    dt[20:40] = 40.0                                       # exp(-640): everything before is forgotten
    dt[60:90] = 0.05
    dt[100] = 1e-30
    d['dt'], d['bias'] = dt.to(dtype).to(_dev()), torch.zeros(2, device=_dev())
    i64 = {k: v.cpu().double() for k, v in d.items()}
    ref = _scan_reference(i64, off, [150], False)
    y, hT, *_ = _outputs(ops, d, (off_d, len_d, 150), softplus=False)
    out = 500 + (2 ** 16 if dtype == torch.bfloat16 else 0)
    _close(y, ref['y'], ref['ya'], out, 'y')
    _close(hT, ref['hT'], ref['ha'], 500, 'hT')
    g = ops.ssm_scan_backward(d['dy'], d['x'], d['dt'], d['A'], d['B'], d['C'], off_d, len_d, 150, D=d['D'], dt_bias=d['bias'], h0=d['h0'], dhT=d['dhT'])
    for name, got, terms in (('x', g.dx, out), ('B', g.dB, 2 * out), ('C', g.dC, 2 * out), ('raw', g.ddt, 1000), ('A', g.dA, 1000), ('h0', g.dh0, 500)):
        assert torch.isfinite(got).all(), name
        _close(got, ref['grads'][name], ref['size'][name], terms, name)


def test_ssm_scan_gradients_against_differences():
    # d(sum of y * dy + hT * dhT) along random directions, by central differences of the f32 forward pass evaluated in its own arithmetic: the
    # difference quotient of step h is off by h^2 times the third derivative and by the forward's rounding over h; with h = 2^-7 and values
    # of order one both stay below 2 % of the directional derivative's magnitude
    from dotaclient_amd import ops
    off_d, len_d, rows, off, d = _scan_inputs(13, [90, 40], 0, 2, 32, 1, 16, torch.float32, 0)
    seqs = (off_d, len_d, 90)
    def value(**change):
        e = dict(d, **change)
        y, hT = ops.ssm_scan(e['x'], e['dt'], e['A'], e['B'], e['C'], *seqs, D=e['D'], dt_bias=e['bias'], h0=e['h0'], softplus=True)
        return float((y.double() * d['dy'].double()).sum() + (hT.double() * d['dhT'].double()).sum())
    g = ops.ssm_scan_backward(d['dy'], d['x'], d['dt'], d['A'], d['B'], d['C'], *seqs, D=d['D'], dt_bias=d['bias'], h0=d['h0'], softplus=True, dhT=d['dhT'])
    gen = torch.Generator().manual_seed(3)
    for key, grad in (('x', g.dx), ('dt', g.ddt), ('A', g.dA), ('B', g.dB), ('C', g.dC), ('D', g.dD), ('bias', g.ddt_bias), ('h0', g.dh0)):
        direction = torch.randn(d[key].shape, generator=gen).to(_dev())
        h = 2.0 ** -7
        slope = (value(**{key: (d[key] + h * direction).contiguous()}) - value(**{key: (d[key] - h * direction).contiguous()})) / (2 * h)
        want = float((grad.double() * direction.double()).sum())
        scale = float((grad.double().abs() * direction.double().abs()).sum())
        assert abs(slope - want) <= 0.02 * scale, (key, slope, want, scale)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('H,P,G,N', [(8, 64, 1, 64), (3, 7, 3, 5), (4, 100, 2, 128)])
def test_ssm_step_against_the_definition(H, P, G, N, dtype):
    from dotaclient_amd import ops
    dev = _dev()
    n = 5
    _, _, rows, off, d = _scan_inputs(14, [1] * n, 0, H, P, G, N, dtype, 3)
    i64 = {k: v.cpu().double() for k, v in d.items()}
    ref = _scan_reference(i64, list(range(n)), [1] * n, True)
    kw = dict(D=d['D'], dt_bias=d['bias'], softplus=True)
    y, hT = ops.ssm_step(d['x'], d['dt'], d['A'], d['B'], d['C'], h0=d['h0'], **kw)
    # N products in lanes of at most 4 and a tree of sixteen, exp and softplus a few steps each
    _close(y, ref['y'], ref['ya'], N + 32, 'y')
    _close(hT, ref['hT'], ref['ha'], 32, 'hT')
    h = d['h0'].clone()
    y2, h2 = ops.ssm_step(d['x'], d['dt'], d['A'], d['B'], d['C'], h0=h, hT=h, **kw)
    assert h2.data_ptr() == h.data_ptr() and torch.equal(h2, hT) and torch.equal(y2, y)
    y3, h3 = ops.ssm_step(d['x'], d['dt'], d['A'], d['B'], d['C'], **kw)
    zero = torch.zeros_like(d['h0'])
    y4, h4 = ops.ssm_step(d['x'], d['dt'], d['A'], d['B'], d['C'], h0=zero, **kw)
    assert torch.equal(y3, y4) and torch.equal(h3, h4)


def test_nothing_to_do_is_done():
    from dotaclient_amd import ops
    dev = _dev()
    f = lambda *s: torch.zeros(*s, device=dev)                                         # noqa: E731
    none = torch.zeros(0, dtype=torch.int64, device=dev), torch.zeros(0, dtype=torch.int32, device=dev), 0
    empty = torch.zeros(2, dtype=torch.int64, device=dev), torch.zeros(2, dtype=torch.int32, device=dev), 0
    h0, st = torch.randn(2, 2, 8, 4, device=dev), torch.randn(2, 2, 16, device=dev)
    for seqs, n in ((none, 0), (empty, 2)):
        for rows in (0, 3):
            y, hT = ops.ssm_scan(f(rows, 2, 8), f(rows, 2), f(2), f(rows, 1, 4), f(rows, 1, 4), *seqs, h0=h0[:n].contiguous())
            assert y.shape == (rows, 2, 8) and torch.equal(hT, h0[:n])
            g = ops.ssm_scan_backward(f(rows, 2, 8), f(rows, 2, 8), f(rows, 2), f(2), f(rows, 1, 4), f(rows, 1, 4), *seqs, D=f(2), h0=h0[:n].contiguous(),
                                      dhT=h0[:n].contiguous())
            assert torch.equal(g.dh0, h0[:n]) and not g.dA.any() and not g.dD.any()
            y, so = ops.causal_conv(f(rows, 16), f(16, 3), f(16), *seqs, state=st[:n].contiguous())
            assert torch.equal(so, st[:n])
            _, dw, db, ds = ops.causal_conv_backward(f(rows, 16), f(rows, 16), f(16, 3), f(16), *seqs, state=st[:n].contiguous(), dstate_out=st[:n].contiguous())
            assert torch.equal(ds, st[:n]) and not dw.any() and not db.any()
    r, x = ops.block_norm(f(0, 8), f(0, 8), f(8), w_pre=f(8))
    assert r.shape == (0, 8) and x.shape == (0, 8)
    out = ops.block_norm_backward(f(0, 8), f(0, 8), f(0, 8), f(0, 8), f(8), w_pre=f(8))
    assert not out[2].any() and not out[5].any()
    y, h = ops.ssm_step(f(0, 2, 8), f(0, 2), f(2), f(0, 1, 4), f(0, 1, 4))
    assert h.shape == (0, 2, 8, 4)


# ------------------------------------------------------------------------------------------------------------- a block of them


def _block_weights(seed, D, inner, H, N, K):
    g = torch.Generator().manual_seed(seed)
    w = dict(w_in=_rand(g, D, 2 * inner + 2 * N + H) * D ** -0.5, w_conv=_rand(g, inner + 2 * N, K) * 0.5, b_conv=0.1 * _rand(g, inner + 2 * N),
             A=-(1 + 3 * torch.rand(H, generator=g, dtype=torch.float64)), Dk=_rand(g, H), dt_bias=-2 + _rand(g, H), w_out=_rand(g, inner, D) * inner ** -0.5,
             w_post=1 + 0.1 * _rand(g, D), scale=0.5 + 0.1 * _rand(g, D), w_pre=1 + 0.1 * _rand(g, D))
    return w


def _block_forward(ops, w, x, r, seqs, H, N, state=None, h0=None):
    """x (normed input), r (residual) [rows, D] -> (r', x'), the carried states and what the backward pass needs."""
    inner = w['w_out'].shape[0]
    z_xbc = x @ w['w_in']
    gate, xbc_in, dt = z_xbc[:, :inner], z_xbc[:, inner:2 * inner + 2 * N], z_xbc[:, 2 * inner + 2 * N:]
    if seqs is None:
        xbc, state = ops.causal_conv_step(xbc_in, state, w['w_conv'], w['b_conv'])
    else:
        xbc, state = ops.causal_conv(xbc_in, w['w_conv'], w['b_conv'], *seqs, state=state)
    v = (xbc[:, :inner].unflatten(1, (H, -1)), dt, w['A'], xbc[:, inner:inner + N].unflatten(1, (1, N)), xbc[:, inner + N:].unflatten(1, (1, N)))
    kw = dict(D=w['Dk'], dt_bias=w['dt_bias'], h0=h0, softplus=True)
    y, h = ops.ssm_step(*v, **kw) if seqs is None else ops.ssm_scan(*v, *seqs, **kw)
    y = y.flatten(1)
    gated = y * torch.nn.functional.silu(gate)
    out = gated @ w['w_out']
    r2, x2 = ops.block_norm(out, r, w['w_post'], scale=w['scale'], w_pre=w['w_pre'])
    return r2, x2, state, h, dict(x=x, gate=gate, xbc_in=xbc_in, v=v, y=y, gated=gated, out=out, r=r, kw=kw)


def _block64(w, x, r, lens, H, N, dr, dx):
    """The same block in f64 with autograd: outputs and the gradients of every weight."""
    leaves = {k: v.clone().requires_grad_(True) for k, v in w.items()}
    inner, K = w['w_out'].shape[0], w['w_conv'].shape[1]
    zx = x @ leaves['w_in']
    gate, xbc, dt = zx[:, :inner], zx[:, inner:2 * inner + 2 * N], zx[:, 2 * inner + 2 * N:]
    ys, o = [], 0
    for m in lens:
        ext = torch.cat([xbc.new_zeros(K - 1, xbc.shape[1]), xbc[o:o + m]])
        c = torch.nn.functional.silu(sum(leaves['w_conv'][:, k] * ext[k:k + m] for k in range(K)) + leaves['b_conv'])
        d = torch.nn.functional.softplus(dt[o:o + m] + leaves['dt_bias'])
        y, _ = _scan64(c[:, :inner].unflatten(1, (H, -1)), d, d * leaves['A'], c[:, inner:inner + N][:, None], c[:, inner + N:][:, None], leaves['Dk'],
                       xbc.new_zeros(1, H, inner // H, N), [0], [m])
        ys.append(y.flatten(1))
        o += m
    out = (torch.cat(ys) * torch.nn.functional.silu(gate)) @ leaves['w_out']
    r2, x2 = _norm64(out, r, leaves['w_post'], None, leaves['scale'], leaves['w_pre'], 1e-5)
    keys = list(leaves)
    grads = torch.autograd.grad((r2 * dr).sum() + (x2 * dx).sum(), [leaves[k] for k in keys])
    return r2.detach(), x2.detach(), dict(zip(keys, grads))


def test_a_block_of_them_trains_and_steps():
    # norm -> projection -> convolution -> scan -> gate -> projection -> norm, scale, residual -> norm: its outputs, its weights' gradients and their
    # clipping against f64, and the same rows one at a time with the states carried.  Relative to each tensor's norm: the longest way through the
    # block has some 2^7 roundings of f32 one after the other or summed up, and no cancellation beyond the sums' own: 2^9 * 2^-24 = 3e-5.
    from dotaclient_amd import ops
    dev = _dev()
    D, H, P, N, K, lens = 32, 4, 16, 16, 4, [37, 70, 5]
    inner, rows = H * P, sum(lens)
    w64 = _block_weights(21, D, inner, H, N, K)
    w = {k: v.float().to(dev) for k, v in w64.items()}
    g = torch.Generator().manual_seed(22)
    x64, r64, dr64, dx64 = (_rand(g, rows, D).float().double() for _ in range(4))
    off_d, len_d, _, off = _packed(lens)
    seqs = (off_d, len_d, max(lens))
    r2, x2, state, h, s = _block_forward(ops, w, x64.float().to(dev), r64.float().to(dev), seqs, H, N)
    w32 = {k: v.cpu().double() for k, v in w.items()}
    rw, xw, gw = _block64(w32, x64, r64, lens, H, N, dr64, dx64)
    near = lambda a, b, what, tol=3e-5: (float((a.cpu().double() - b).norm()) <= tol * float(b.norm())) or pytest.fail(     # noqa: E731
        '%s: %.2e' % (what, float((a.cpu().double() - b).norm() / b.norm())))
    near(r2, rw, 'r'), near(x2, xw, 'x')
    # backward, by the operators' own gradients
    dout, dres, dw_post, _, dscale, dw_pre = ops.block_norm_backward(dr64.float().to(dev), dx64.float().to(dev), s['out'], s['r'], w['w_post'],
                                                                     scale=w['scale'], w_pre=w['w_pre'])
    dgated = dout @ w['w_out'].t()
    sg = torch.sigmoid(s['gate'])
    dy, dgate = dgated * s['gate'] * sg, dgated * s['y'] * sg * (1 + s['gate'] * (1 - sg))
    # the gradients of x, B and C go to the columns of one tensor, as the convolution wants them
    dxbc = torch.empty(rows, inner + 2 * N, device=dev)
    sc = ops.ssm_scan_backward(dy.unflatten(1, (H, P)), *s['v'], *seqs, **s['kw'], dx=dxbc[:, :inner].unflatten(1, (H, P)),
                               dB=dxbc[:, inner:inner + N].unflatten(1, (1, N)), dC=dxbc[:, inner + N:].unflatten(1, (1, N)))
    dconv, dw_conv, db_conv, _ = ops.causal_conv_backward(dxbc, s['xbc_in'], w['w_conv'], w['b_conv'], *seqs)
    dzx = torch.cat([dgate, dconv, sc.ddt], 1)
    grads = dict(w_in=s['x'].t() @ dzx, w_conv=dw_conv, b_conv=db_conv, A=sc.dA, Dk=sc.dD, dt_bias=sc.ddt_bias, w_out=s['gated'].t() @ dout, w_post=dw_post,
                 scale=dscale, w_pre=dw_pre)
    for k in gw:
        near(grads[k], gw[k], 'gradient of ' + k, 1e-4)
    keys = list(gw)
    clip = ops.GradNormClip([grads[k].contiguous() for k in keys])
    total, norms = clip(0.5)
    want = torch.stack([gw[k].norm() for k in keys])
    near(norms, want, 'norms', 1e-4), near(total[None], want.norm()[None], 'total', 1e-4)
    near(torch.cat([t.flatten() for t in clip._tensors[0]]), torch.cat([gw[k].flatten() for k in keys]) * (0.5 / float(want.norm())), 'clipped', 2e-4)
    # one row at a time, every sequence its own hero
    n = len(lens)
    st, hs = torch.zeros(n, K - 1, inner + 2 * N, device=dev), torch.zeros(n, H, P, N, device=dev)
    xd, rd = x64.float().to(dev), r64.float().to(dev)
    for t in range(max(lens)):
        at = torch.tensor([o + min(t, m - 1) for o, m in zip(off, lens)], device=dev)
        live = torch.tensor([t < m for m in lens], device=dev)
        rs, xs, st2, hs2, _ = _block_forward(ops, w, xd[at], rd[at], None, H, N, st, hs)
        st, hs = torch.where(live[:, None, None], st2, st), torch.where(live[:, None, None, None], hs2, hs)
        for k in range(n):
            if bool(live[k]):
                near(rs[k], rw[int(at[k])], 'step %d of sequence %d' % (t, k))
    near(hs, h.cpu().double(), 'carried state'), near(st, state.cpu().double(), 'carried convolution state')
    # a sequence in two pieces with the states carried between them
    cut = [20, 33, 2]
    first = torch.tensor(cut, dtype=torch.int32, device=dev)
    ra, _, sa, ha, _ = _block_forward(ops, w, xd, rd, (off_d, first, max(cut)), H, N)
    rb, _, sb, hb, _ = _block_forward(ops, w, xd, rd, (off_d + first, len_d - first, max(lens)), H, N, sa, ha)
    for k, (o, m) in enumerate(zip(off, lens)):
        near(torch.cat([ra[o:o + cut[k]], rb[o + cut[k]:o + m]]), rw[o:o + m], 'pieces of sequence %d' % k)
    near(hb, h.cpu().double(), 'state behind the pieces'), near(sb, state.cpu().double(), 'convolution state behind the pieces')


# ------------------------------------------------------------------------------------------------------- streams, graphs, addresses


def _all_calls(ops, d, conv, norm, clip):
    seqs = d['seqs']
    out = _outputs(ops, d, seqs)
    y, so = ops.causal_conv(conv['x'], conv['w'], conv['b'], *seqs, state=conv['state'])
    out += [y, so] + list(ops.causal_conv_backward(conv['dy'], conv['x'], conv['w'], conv['b'], *seqs, state=conv['state']))
    out += list(ops.block_norm(norm['y'], norm['r'], norm['wp'], gate=norm['z'], scale=norm['s'], w_pre=norm['wq']))
    out += list(ops.block_norm_backward(norm['dr'], norm['dx'], norm['y'], norm['r'], norm['wp'], gate=norm['z'], scale=norm['s'], w_pre=norm['wq']))
    total, norms = clip(0.5)
    return [t for t in out if t is not None] + [total, norms] + clip._tensors[1]


def _call_inputs(seed):
    dev = _dev()
    g = torch.Generator().manual_seed(seed)
    lens = [200, 3, 77]
    off_d, len_d, rows, off, d = _scan_inputs(seed, lens, 0, 4, 32, 2, 16, torch.bfloat16, 0)
    d['seqs'] = (off_d, len_d, 200)
    f = lambda *s: _rand(g, *s).float().to(dev)                                        # noqa: E731
    conv = dict(x=f(rows, 40), dy=f(rows, 40), w=f(40, 4), b=f(40), state=f(3, 3, 40))
    norm = dict(y=f(rows, 100), r=f(rows, 100), z=f(rows, 100), dr=f(rows, 100), dx=f(rows, 100), wp=f(100), s=f(100), wq=f(100))
    grads = [f(1000), f(7), f(40000)]
    return d, conv, norm, grads


def test_calls_on_two_streams_and_in_two_graphs_share_nothing():
    from dotaclient_amd import ops
    inputs = [_call_inputs(s) for s in (31, 32)]
    clips = [ops.GradNormClip(i[3], [torch.empty_like(t) for t in i[3]]) for i in inputs]
    # two of them on the same gradients with outputs of their own
    want = [[t.clone() for t in _all_calls(ops, *i[:3], c)] for i, c in zip(inputs, clips)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = [None, None]
        for k, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got[k] = _all_calls(ops, *inputs[k][:3], clips[k])
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    graphs, outs = [], []
    for k, s in enumerate(streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(_all_calls(ops, *inputs[k][:3], clips[k]))
        graphs.append(g)
    for turn in range(3):
        # new values in the same buffers, eager work of the program's own in between
        for k in range(2):
            fresh = _call_inputs(40 + 2 * turn + k)
            for old, new in zip(inputs[k][:3], fresh[:3]):
                for key in old:
                    if torch.is_tensor(old[key]):
                        old[key].copy_(new[key])
            for old, new in zip(inputs[k][3], fresh[3]):
                old.copy_(new)
        want = [[t.clone() for t in _all_calls(ops, *i[:3], c)] for i, c in zip(inputs, clips)]
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, outs):
            assert all(torch.equal(x, y) for x, y in zip(a, b)), turn


def test_rows_far_apart():
    # rows 2^22 elements from each other: offsets beyond 2^31 elements
    from dotaclient_amd import ops
    dev = _dev()
    rows, ld = 600, 1 << 22
    lens = [300, 299]
    off_d, len_d, _, off, d = _scan_inputs(51, lens, 0, 2, 16, 1, 16, torch.bfloat16, 0)
    wide = torch.empty(rows * ld, dtype=torch.bfloat16, device=dev).view(rows, ld)
    xs = wide[:599, ld - 32:].unflatten(1, (2, 16))
    xs.copy_(d['x'])
    near = _outputs(ops, d, (off_d, len_d, 300))
    far = _outputs(ops, dict(d, x=xs), (off_d, len_d, 300))
    assert all(torch.equal(a, b) for a, b in zip(near, far))
    ys = wide[:599, 64:96].unflatten(1, (2, 16))
    ops.ssm_scan(d['x'], d['dt'], d['A'], d['B'], d['C'], off_d, len_d, 300, D=d['D'], dt_bias=d['bias'], h0=d['h0'], softplus=True, y=ys)
    assert torch.equal(ys, near[0])
    flat = xs.flatten(1)
    w = torch.randn(32, 4, device=dev)
    assert torch.equal(ops.causal_conv(flat, w, None, off_d, len_d, 300)[0], ops.causal_conv(d['x'].flatten(1), w, None, off_d, len_d, 300)[0])
    wp = torch.randn(32, device=dev)
    assert torch.equal(ops.block_norm(flat, flat, wp)[0], ops.block_norm(d['x'].flatten(1).contiguous(), d['x'].flatten(1).contiguous(), wp)[0])
    # one row of step sizes for all of them, not copied (raw ones: heads whose sizes are negative grow beyond every number, NaN in both)
    one = d['dt'][:1].expand(599, -1)
    a = ops.ssm_scan(d['x'], one, d['A'], d['B'], d['C'], off_d, len_d, 300)[0]
    b = ops.ssm_scan(d['x'], one.contiguous(), d['A'], d['B'], d['C'], off_d, len_d, 300)[0]
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0.0), b.nan_to_num(0.0))
