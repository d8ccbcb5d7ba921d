"""Rotary positions with several axes (ops.rotary_axes) and the norms of queries and keys with the rotation in the same pass
(ops.qk_norm_rotary), against the definition in 64 bits.

Tolerances.  A value stored in type T is off by at most eps(T) / 2 of itself.  Before that, in float32 (u = 2^-24):
 * cos and sin: the reduced angle is rounded once (u / 2 * pi / 4), the series' terms round a few times: 2 u; the rotation's two
   products and one sum: together at most 6 u (|a| + |b|) for the pair (a, b).
 * the norm: a sum of dh squares is off by at most (dh - 1) u of itself, its root by half of that; rsqrt, the products and the gain
   another 10 u: (dh / 2 + 16) u (|za| + |zb|) with the rotation.
 * dx = r (t - xh mean(t xh)): r twice, the sum of dh terms of mixed signs: (2 dh + 32) u r (T + |xh| mean(T |xh|)), T = |gain| (|dya| + |dyb|).
 * dgain: a sum over the n tokens of terms that are themselves off by (dh / 2 + 24) u: (n + dh / 2 + 24) u sum(T' |xh|)."""
import ctypes

import pytest
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2 if dtype == torch.bfloat16 else 0.0


def angles(positions, inv_freq, sections):
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    return positions.double()[:, axis] * inv_freq[None]


def turn(x, theta, interleaved):
    """[n, h, dh] float64"""
    p = theta.shape[1]
    c, s = theta.cos()[:, None], theta.sin()[:, None]
    y = x.clone()
    ia = torch.arange(p) * 2 if interleaved else torch.arange(p)
    ib = ia + 1 if interleaved else ia + p
    a, b = x[..., ia], x[..., ib]
    y = y.index_copy(2, ia, a * c - b * s).index_copy(2, ib, a * s + b * c)
    return y


def pair_size(x, p, interleaved):
    """|a| + |b| at both channels of a pair, |x| at the others"""
    ia = torch.arange(p) * 2 if interleaved else torch.arange(p)
    ib = ia + 1 if interleaved else ia + p
    m = x.abs()
    both = m[..., ia] + m[..., ib]
    return m.index_copy(2, ia, both).index_copy(2, ib, both)


def within(got, want, tol, what):
    got = got.detach().double().cpu()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f'{what}: {int(bad.sum())} of {bad.numel()} values, worst {((got - want).abs() / tol.clamp_min(1e-300)).max():.3g} of the tolerance'


def make_positions(n, axes, kind, g):
    if kind == torch.float32:
        return torch.randn(n, axes, generator=g) * 300
    top = (1 << 40) if kind == torch.int64 else 500
    return torch.randint(-top, top, (n, axes), generator=g).to(kind)


SHAPES = [  # n, h, dh, sections, interleaved, dtype, positions' type, spare heads in a row
    (1, 16, 32, (4, 6, 6), False, torch.bfloat16, torch.int32, 0),
    (1, 1, 2, (1,), True, torch.float32, torch.int32, 0),
    (3, 1, 512, (100, 100, 56), False, torch.bfloat16, torch.int32, 1),
    (63, 16, 16, (4, 4), False, torch.bfloat16, torch.int32, 8),
    (2049, 16, 16, (4, 4), False, torch.float32, torch.int32, 8),
    (4097, 8, 16, (8,), True, torch.bfloat16, torch.int64, 0),
    (257, 7, 40, (4, 6, 6), True, torch.float32, torch.int64, 0),
    (257, 7, 40, (4, 6, 6), False, torch.float32, torch.float32, 3),
    (100, 5, 24, (3, 4, 1, 2), False, torch.bfloat16, torch.int32, 0),          # the halves meet at no multiple of 4
    (100, 5, 24, (3, 4), False, torch.float32, torch.int32, 0),
    (129, 3, 10, (2, 2), False, torch.bfloat16, torch.int32, 0),                # no whole units of 8 channels
    (129, 3, 10, (3, 2), True, torch.float32, torch.float32, 0),
    (130, 3, 7, (2, 1), False, torch.float32, torch.int32, 0),
    (50, 200, 64, (10, 10, 12), False, torch.bfloat16, torch.int32, 0),         # more heads than a workgroup holds
    (33, 48, 96, (16, 16, 16), True, torch.bfloat16, torch.int32, 0),
    (1000, 20, 72, (12, 12, 12), False, torch.float32, torch.int32, 0),
]


def build(n, h, dh, sections, interleaved, dtype, kind, spare, seed=0):
    from tmae_amd import ops
    g = torch.Generator().manual_seed(seed)
    wide = (torch.randn(n, h + spare, dh, generator=g) * 1.5).to(dtype)
    pos = make_positions(n, len(sections), kind, g)
    return wide, pos, ops.rotary_freqs(sections, 100.0), torch.randn(n, h, dh, generator=g).to(dtype), g


# --------------------------------------------------------------------------------------------------------------- the CPU

def test_frequencies_are_a_ladder_for_each_axis():
    from tmae_amd import ops
    f = ops.rotary_freqs((2, 3), 100.0)
    assert f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 1.0, 100.0 ** (-1 / 3), 100.0 ** (-2 / 3)], dtype=torch.float64), rtol=1e-14)
    for bad in ((), (0,), (2, -1)):
        with pytest.raises(ValueError):
            ops.rotary_freqs(bad)
    with pytest.raises(ValueError):
        ops.rotary_freqs((2,), 0.0)


def test_refusals():
    from tmae_amd import ops
    x, pos, f = torch.zeros(4, 6, 16), torch.zeros(4, 2, dtype=torch.int32), ops.rotary_freqs((4, 4))
    gain = torch.ones(16)

    def refused(kind, match, fn, *a, **k):
        with pytest.raises(kind, match=match):
            fn(*a, **k)
    for fn, gains in ((ops.rotary_axes, ()), (ops.qk_norm_rotary, (gain, gain))):
        def call(x=x, pos=pos, f=f, sec=(4, 4), fn=fn, gains=gains, **k):
            return fn(x, *gains, pos, f, sec, **k)
        refused(RuntimeError, 'GPU only', call)
        refused(ValueError, r'\[tokens, heads, channels\]', call, x=x[0])
        refused(TypeError, 'float32 / bfloat16', call, x=x.half())
        refused(ValueError, 'sections', call, sec=(4, 5), f=ops.rotary_freqs((4, 5)))
        refused(ValueError, 'sections', call, sec=(), pos=pos[:, :0])
        refused(ValueError, 'sections', call, sec=(4, 0))
        refused(ValueError, 'sections', call, sec=(1,) * 5)
        refused(ValueError, 'positions', call, pos=pos[:3])
        refused(ValueError, 'positions', call, pos=pos[:, :1])
        refused(TypeError, 'positions', call, pos=pos.double())
        refused(ValueError, 'inv_freq', call, f=f.float())
        refused(ValueError, 'inv_freq', call, f=f[:5])
        refused(ValueError, 'no gradient', call, f=f.clone().requires_grad_())
    refused(ValueError, '512', ops.rotary_axes, torch.zeros(4, 1, 520), pos, f, (4, 4))

    def norm(q=gain, k=gain, x=x, **kw):
        return ops.qk_norm_rotary(x, q, k, pos, f, (4, 4), **kw)
    refused(ValueError, 'q_heads', norm, q_heads=7)
    refused(ValueError, 'q_heads', norm, q_heads=-1)
    refused(ValueError, 'q_heads', norm, x=x[:, :5])
    refused(ValueError, 'eps', norm, eps=-1.0)
    refused(ValueError, 'eps', norm, eps=float('nan'))
    refused(TypeError, 'q_gain', norm, q=gain.bfloat16())
    refused(ValueError, 'k_gain', norm, k=gain[:8])
    refused(ValueError, 'one kind', norm, q=torch.ones(3, 16))
    refused(ValueError, 'q_gain', norm, q=torch.ones(4, 16), k=torch.ones(3, 16))


def test_c_entries_refuse_bad_arguments():
    """The host's checks come before any launch: bad calls return an error code without a GPU."""
    from tmae_amd._lib import lib
    sec = (ctypes.c_int32 * 2)(4, 4)
    one = ctypes.c_void_p(16)

    def rot(x=one, ldx=96, hpx=16, dtype=1, n=4, h=6, dh=16, pos=one, kind=0, ldpos=2, f=one, sec=sec, axes=2, y=one):
        return lib.tmae_rotary_axes(x, ldx, hpx, dtype, n, h, dh, pos, kind, ldpos, f, sec, axes, 0, 0, y, None)
    assert rot(n=0) == 0
    assert rot(dtype=2) == -3
    for bad in (dict(x=None), dict(pos=None), dict(f=None), dict(y=None), dict(sec=None), dict(n=-1), dict(h=0), dict(h=65536), dict(dh=0),
                dict(dh=15), dict(dh=520), dict(axes=0), dict(axes=5), dict(kind=3), dict(kind=-1), dict(ldpos=1), dict(ldx=-1),
                dict(sec=(ctypes.c_int32 * 2)(8, 1)), dict(sec=(ctypes.c_int32 * 2)(0, 1)), dict(sec=(ctypes.c_int32 * 2)(2 ** 31 - 1, 2 ** 31 - 1))):
        assert rot(**bad) == -1, bad

    def bwd(q_heads=3, eps=1e-6, dq=one, ws=one, ws_bytes=0, dy=one):
        return lib.tmae_qk_norm_rotary_bwd(one, 96, 16, dy, 1, 4, 6, q_heads, 16, one, one, 0, eps, one, 0, 2, one, sec, 2, 0, one, dq, None,
                                           ws, ws_bytes, None)
    assert bwd(q_heads=7) == -1 and bwd(q_heads=-1) == -1 and bwd(eps=-1.0) == -1 and bwd(eps=float('nan')) == -1 and bwd(dy=None) == -1
    need = lib.tmae_qk_norm_rotary_bwd_workspace(4, 6, 16, 8, 0)
    assert need > 0 and bwd(ws_bytes=need - 1) == -2 and bwd(ws=None, ws_bytes=need) == -2
    assert lib.tmae_qk_norm_rotary_bwd_workspace(0, 6, 16, 8, 0) == 0


# --------------------------------------------------------------------------------------------------------------- the GPU

@pytest.mark.gpu
@pytest.mark.parametrize('case', SHAPES, ids=lambda c: f'{c[0]}x{c[1]}x{c[2]}')
def test_rotation_and_its_gradient(case):
    from tmae_amd import ops
    n, h, dh, sections, inter, dtype, kind, spare = case
    wide, pos, f, dy, _ = build(*case)
    theta, p = angles(pos, f, sections), sum(sections)
    x = wide[:, :h].double()
    x_gpu = wide.cuda()[:, :h].detach().requires_grad_()
    y = ops.rotary_axes(x_gpu, pos.cuda(), f.cuda(), sections, interleaved=inter)
    dx, = torch.autograd.grad(y, x_gpu, dy.cuda())
    assert y.dtype == dtype and y.shape == (n, h, dh) and y.is_contiguous()
    want = turn(x, theta, inter)
    within(y, want, half_step(dtype) * want.abs() + 6 * U * pair_size(x, p, inter), 'y')
    want = turn(dy.double(), -theta, inter)
    within(dx, want, half_step(dtype) * want.abs() + 6 * U * pair_size(dy.double(), p, inter), 'dx')
    assert torch.equal(y[..., 2 * p:].cpu(), wide[:, :h, 2 * p:])                       # what does not turn passes as it is
    with torch.no_grad():
        assert torch.equal(ops.rotary_axes(x_gpu, pos.cuda(), f.cuda(), sections, interleaved=inter), y)
        assert torch.equal(ops.rotary_axes(dy.cuda(), pos.cuda(), f.cuda(), sections, interleaved=inter, inverse=True), dx)


def norm_reference(x, gains, theta, inter, eps):
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    return turn(x * r * gains, theta, inter)


@pytest.mark.gpu
@pytest.mark.parametrize('per_head', [False, True])
@pytest.mark.parametrize('case', SHAPES, ids=lambda c: f'{c[0]}x{c[1]}x{c[2]}')
def test_norm_with_rotation_and_its_gradients(case, per_head):
    from tmae_amd import ops
    n, h, dh, sections, inter, dtype, kind, spare = case
    wide, pos, f, dy, g = build(*case, seed=1)
    hq, eps = (h + 1) // 2, 1e-5
    gq, gk = ((1 + 0.3 * torch.randn(*(([k] if per_head else []) + [dh]), generator=g)) for k in (hq, h - hq))
    if per_head and h == hq:
        gk = None
    theta, p = angles(pos, f, sections), sum(sections)
    x = wide[:, :h].double()
    gains = torch.cat([gq.double().expand(hq, dh), torch.zeros(0, dh) if gk is None else gk.double().expand(h - hq, dh)])
    x_gpu = wide.cuda()[:, :h].detach().requires_grad_()
    gq_gpu = gq.cuda().requires_grad_()
    gk_gpu = None if gk is None else gk.cuda().requires_grad_()
    y = ops.qk_norm_rotary(x_gpu, gq_gpu, gk_gpu, pos.cuda(), f.cuda(), sections, q_heads=hq, eps=eps, interleaved=inter)
    want = norm_reference(x, gains, theta, inter, eps)
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    within(y, want, half_step(dtype) * want.abs() + (dh / 2 + 16) * U * pair_size(x * r * gains, p, inter), 'y')
    leaves = [x_gpu, gq_gpu] + ([] if gk is None else [gk_gpu])
    got = torch.autograd.grad(y, leaves, dy.cuda())
    # the formula
    xh, dz = x * r, turn(dy.double(), -theta, inter)
    t = dz * gains
    dx = r * (t - xh * (t * xh).mean(-1, keepdim=True))
    size = pair_size(dy.double(), p, inter)
    T = size * gains.abs()
    within(got[0], dx, half_step(dtype) * dx.abs() + (2 * dh + 32) * U * r * (T + xh.abs() * (T * xh.abs()).mean(-1, keepdim=True)), 'dx')
    terms, sizes = dz * xh, size * xh.abs()
    for i, (lo, hi) in enumerate([(0, hq), (hq, h)][:len(got) - 1]):
        want, tol = terms[:, lo:hi].sum(0), (n + dh / 2 + 24) * U * sizes[:, lo:hi].sum(0)
        if not per_head:
            want, tol = want.sum(0), tol.sum(0) * (hi - lo if hi > lo else 1)
        within(got[1 + i], want, tol + half_step(torch.float32) + U * want.abs(), f'dgain {i}')
    # differences along a direction, in 64 bits
    step = 1e-6
    ux, ug = torch.randn(x.shape, generator=g).double(), torch.randn(gains.shape, generator=g).double()
    if not per_head:
        ug = torch.cat([ug[:1].expand(hq, dh), ug[-1:].expand(h - hq, dh)])
    lo, hi = (((norm_reference(x + k * step * ux, gains + k * step * ug, theta, inter, eps)) * dy.double()).sum() for k in (-1, 1))
    along = (dx * ux).sum() + (terms.sum(0) * ug).sum()
    scale = (T * r * ux.abs()).sum() + (sizes.sum(0) * ug.abs()).sum()
    assert abs((hi - lo) / (2 * step) - along) <= 1e-6 * scale


@pytest.mark.gpu
def test_no_tokens_and_no_gains():
    from tmae_amd import ops
    f = ops.rotary_freqs((4, 4), device='cuda')
    x, pos = torch.zeros(0, 4, 16, device='cuda', requires_grad=True), torch.zeros(0, 2, dtype=torch.int32, device='cuda')
    gain = torch.ones(16, device='cuda', requires_grad=True)
    assert ops.rotary_axes(x, pos, f, (4, 4)).shape == (0, 4, 16)
    y = ops.qk_norm_rotary(x, gain, gain, pos, f, (4, 4))
    dx, dg = torch.autograd.grad(y, (x, gain), torch.zeros_like(y))
    assert dx.shape == (0, 4, 16) and torch.equal(dg, torch.zeros_like(gain))
    x = torch.randn(300, 4, 16, device='cuda')
    pos = torch.randint(0, 99, (300, 2), device='cuda')
    bare, ones = (ops.qk_norm_rotary(x, k, k, pos, f, (4, 4), q_heads=2) for k in (None, gain.detach()))
    assert torch.equal(bare, ones)
    xr = x.clone().requires_grad_()
    dx, = torch.autograd.grad(ops.qk_norm_rotary(xr, None, None, pos, f, (4, 4)), xr, x)
    assert torch.isfinite(dx).all()


@pytest.mark.gpu
@pytest.mark.parametrize('value', [float('nan'), float('inf')])
def test_a_bad_token_stays_alone(value):
    """NaN and infinities of one head of one token reach that head only (of the gains' gradients: its side's)."""
    from tmae_amd import ops
    n, h, dh, sec = 301, 6, 24, (3, 4)
    f = ops.rotary_freqs(sec, device='cuda')
    pos = torch.randint(0, 99, (n, 2), device='cuda')
    for inter in (False, True):
        x = torch.randn(n, h, dh, device='cuda')
        x[17, 2, 5] = value
        gain = torch.ones(dh, device='cuda')
        x.requires_grad_()
        y = ops.qk_norm_rotary(x, gain, gain, pos, f, sec, interleaved=inter)
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        for t in (y, dx, ops.rotary_axes(x, pos, f, sec, interleaved=inter)):
            bad = ~torch.isfinite(t).all(-1)
            assert bad[17, 2] and bad.sum() == 1
    zero = torch.zeros(5, 2, 16, device='cuda', requires_grad=True)
    y = ops.qk_norm_rotary(zero, None, None, torch.zeros(5, 1, dtype=torch.int32, device='cuda'), ops.rotary_freqs((8,), device='cuda'), (8,))
    dx, = torch.autograd.grad(y, zero, torch.ones_like(y))
    assert torch.equal(y, torch.zeros_like(y)) and torch.isfinite(dx).all()


@pytest.mark.gpu
def test_strides_alignment_and_streams():
    """Odd pitches and bases, columns apart, broadcast gradients and positions, a stream of its own: the same bits as the plain call."""
    from tmae_amd import ops
    n, h, dh, sec = 517, 4, 32, (4, 5, 7)
    f = ops.rotary_freqs(sec, device='cuda')
    g = torch.Generator(device='cuda').manual_seed(3)
    gq, gk = (torch.randn(dh, device='cuda', generator=g) for _ in range(2))
    pos = torch.randint(0, 400, (n, 3), device='cuda', dtype=torch.int32, generator=g)
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.randn(n, h, dh, device='cuda', generator=g).to(dtype)
        wide = torch.zeros(n, h * dh + 3, device='cuda', dtype=dtype)
        wide[:, 3:] = x.view(n, -1)
        odd = wide[:, 3:].view(n, h, dh)
        apart = torch.zeros(n, h, 2 * dh, device='cuda', dtype=dtype)
        apart[..., ::2] = x
        turned = x.transpose(0, 1).contiguous().transpose(0, 1)
        wide_pos = torch.zeros(n, 7, device='cuda', dtype=torch.int32)
        wide_pos[:, 2:5] = pos
        outs = [(ops.rotary_axes(v, p, f, sec), ops.qk_norm_rotary(v, gq, gk, p, f, sec))
                for v, p in ((x, pos), (odd, pos), (apart[..., ::2], pos), (turned, wide_pos[:, 2:5]), (x, pos.t().contiguous().t()))]
        for a, b in outs[1:]:
            assert torch.equal(a, outs[0][0])
            assert torch.allclose(b.float(), outs[0][1].float(), rtol=2 * torch.finfo(dtype).eps, atol=1e-6)
        # a broadcast gradient
        xr = x.clone().requires_grad_()
        a, = torch.autograd.grad(ops.qk_norm_rotary(xr, gq, gk, pos, f, sec).float().sum(), xr)
        b, = torch.autograd.grad(ops.qk_norm_rotary(xr, gq, gk, pos, f, sec), xr, torch.ones_like(x))
        assert torch.equal(a, b)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y = ops.qk_norm_rotary(x, gq, gk, pos, f, sec)
        side.synchronize()
        assert torch.equal(y, outs[0][1])


@pytest.mark.gpu
def test_gradients_are_the_same_every_time_and_in_a_graph():
    """No order of additions changes from run to run; a captured step replays to the eager result on new inputs."""
    from tmae_amd import ops
    n, h, dh, sec = 9000, 8, 16, (4, 4)
    f = ops.rotary_freqs(sec, device='cuda')
    pos = torch.randint(0, 400, (n, 2), device='cuda', dtype=torch.int32)
    x = torch.randn(n, h, dh, device='cuda').bfloat16().requires_grad_()
    gq, gk = (torch.randn(dh, device='cuda').requires_grad_() for _ in range(2))
    dy = torch.randn(n, h, dh, device='cuda').bfloat16()

    def step(x):
        y = ops.qk_norm_rotary(x, gq, gk, pos, f, sec)
        z = ops.rotary_axes(y, pos, f, sec, inverse=True)
        return (z.detach(), *torch.autograd.grad(z, (x, gq, gk), dy))
    first = step(x)
    assert all(torch.equal(a, b) for a, b in zip(first, step(x)))
    held = x.detach().clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held)
    for k in range(4):
        fresh = torch.randn(n, h, dh, device='cuda').bfloat16().requires_grad_()
        with torch.no_grad():
            held.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step(fresh))), k


@pytest.mark.gpu
def test_a_second_derivative_is_refused():
    from tmae_amd import ops
    x = torch.randn(9, 2, 16, device='cuda', requires_grad=True)
    pos, f = torch.randint(0, 99, (9, 1), device='cuda'), ops.rotary_freqs((8,), device='cuda')
    for y in (ops.rotary_axes(x, pos, f, (8,)), ops.qk_norm_rotary(x, None, None, pos, f, (8,))):
        dx, = torch.autograd.grad(y.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match='once_differentiable'):
            (y.sum() + dx.sum()).backward()


@pytest.mark.gpu
def test_rows_beyond_32_bits():
    """9 M tokens of 8 + 8 heads of 16 in bfloat16, 2^31 elements and more: the last tokens' results are those of the last tokens alone."""
    from tmae_amd import ops
    n, h, dh, sec, last = 9_000_000, 16, 16, (4, 4), 1000
    g = torch.Generator(device='cuda').manual_seed(1)
    x, dy = (torch.randn(n, h, dh, generator=g, device='cuda', dtype=torch.bfloat16) for _ in range(2))
    assert x.numel() > 2 ** 31
    pos = torch.randint(0, 468, (n, 2), generator=g, device='cuda', dtype=torch.int32)
    f = ops.rotary_freqs(sec, device='cuda')
    gain = torch.rand(dh, generator=g, device='cuda') + 0.5

    def run(x, dy, pos):
        x = x.detach().requires_grad_()
        r, y = ops.rotary_axes(x, pos, f, sec), ops.qk_norm_rotary(x, gain, gain, pos, f, sec)
        return [t.detach() for t in (r, y, *torch.autograd.grad(r, x, dy), *torch.autograd.grad(y, x, dy))]
    for a, b in zip(run(x, dy, pos), run(x[-last:], dy[-last:], pos[-last:])):
        assert torch.equal(a[-last:], b)


@pytest.mark.gpu
@pytest.mark.parametrize('value', [float('inf'), -float('inf'), float('nan')])
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('sections,dh,dtype', [((3,), 16, torch.bfloat16), ((2, 3), 24, torch.float32), ((1,), 7, torch.float32), ((3, 4), 24, torch.bfloat16)])
def test_a_bad_value_that_does_not_turn_stays_in_its_channel(sections, dh, dtype, interleaved, value):
    """Channels from 2 P on pass as they are, whatever stands beside them: in rotary_axes, in the gains of qk_norm_rotary, and in the
    gradient that comes back to it."""
    from tmae_amd import ops
    n, h, p = 67, 3, sum(sections)
    f = ops.rotary_freqs(sections, device='cuda')
    g = torch.Generator(device='cuda').manual_seed(dh)
    pos = torch.randint(0, 99, (n, len(sections)), device='cuda', generator=g)
    x = torch.randn(n, h, dh, device='cuda', generator=g).to(dtype)
    clean = ops.rotary_axes(x, pos, f, sections, interleaved=interleaved)
    gain = torch.rand(dh, device='cuda', generator=g) + 0.5
    normed = ops.qk_norm_rotary(x, gain, gain, pos, f, sections, q_heads=h, interleaved=interleaved)

    def others(c):
        return [e for e in range(dh) if e != c]
    for c in range(2 * p, dh):
        bad = x.clone()
        bad[..., c] = value
        leaf = bad.clone().requires_grad_()
        y = ops.rotary_axes(leaf, pos, f, sections, interleaved=interleaved)
        back = ops.rotary_axes(bad, pos, f, sections, interleaved=interleaved, inverse=True)
        dx, = torch.autograd.grad(y, leaf, bad)
        for t in (y, back, dx):
            assert torch.equal(t[..., 2 * p:].isnan(), bad[..., 2 * p:].isnan())
            assert torch.equal(t[..., 2 * p:].nan_to_num(7.0), bad[..., 2 * p:].nan_to_num(7.0))
        assert torch.equal(y[..., others(c)], clean[..., others(c)])
        wrong = gain.clone()
        wrong[c] = value
        y = ops.qk_norm_rotary(x, wrong, wrong, pos, f, sections, q_heads=h, interleaved=interleaved)
        assert torch.equal(y[..., others(c)], normed[..., others(c)])
        leaves = [gain.clone().requires_grad_(), x.clone().requires_grad_()]
        y = ops.qk_norm_rotary(leaves[1], leaves[0], None, pos, f, sections, interleaved=interleaved)
        dg, = torch.autograd.grad(y, leaves[:1], bad)
        assert torch.isfinite(dg[others(c)]).all() and not torch.isfinite(dg[c])


def test_forward_mode_derivatives_are_refused(monkeypatch):
    """None of these operators has one: a tensor with a tangent is an error, with and without recorded gradients, and so is a tangent on
    the gradient that comes back.  (The launches are left out: this is the host's side.)"""
    from torch.autograd import forward_ad
    from tmae_amd import ops
    monkeypatch.setattr(ops, '_need_cuda', lambda t: None)
    monkeypatch.setattr(ops, '_launch', lambda *a: None)
    pos, f, grid = torch.zeros(64, 2, dtype=torch.int32), ops.rotary_freqs((4, 4)), torch.arange(64, dtype=torch.int32)
    gain = torch.ones(16)
    calls = [(lambda t: ops.rotary_axes(t.view(64, 3, 16), pos, f, (4, 4)), (64, 48)),
             (lambda t: ops.qk_norm_rotary(t.view(64, 3, 16), gain, gain, pos, f, (4, 4), q_heads=2), (64, 48)),
             (lambda t: ops.qk_norm_rotary(torch.ones(64, 3, 16), t, gain, pos, f, (4, 4), q_heads=2), (16,)),
             (lambda t: ops.win_attn_dot(t, None, None, grid, grid, 1, 1, 8, 8, False), (64, 48)),
             (lambda t: ops.win_attn_dot(torch.ones(64, 32), t, None, grid, grid, 1, 1, 8, 8, False), (64, 16))]
    for call, shape in calls:
        plain = torch.ones(shape)
        assert call(plain) is not None
        with forward_ad.dual_level():
            assert call(plain) is not None
            for leaf in (plain, plain.clone().requires_grad_()):
                with pytest.raises((RuntimeError, NotImplementedError), match='forward'):
                    call(forward_ad.make_dual(leaf, plain))
                with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError), match='forward'):
                    call(forward_ad.make_dual(leaf, plain))
            leaf = plain.clone().requires_grad_()
            y = call(leaf)
            torch.autograd.grad(y, leaf, torch.ones_like(y), retain_graph=True)
            with pytest.raises((RuntimeError, NotImplementedError), match='forward'):
                torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))


def test_the_pitch_of_one_tokens_positions(monkeypatch):
    """The stride over a single token (or none) says nothing: transposed positions of one token have 1 there."""
    from tmae_amd import ops
    monkeypatch.setattr(ops, '_need_cuda', lambda t: None)
    seen = []
    monkeypatch.setattr(ops, '_launch', lambda entry, dev, *a: seen.append((entry.__name__, a)))
    f, parts = ops.rotary_freqs((4, 5, 7)), [torch.tensor([t], dtype=torch.int32) for t in (3, 1, 4)]
    for n, pos in ((1, torch.stack(parts).t()), (1, torch.stack(parts, 1)), (1, torch.arange(9).view(1, 9)[:, ::4]),
                   (0, torch.zeros(3, 0, dtype=torch.int32).t())):
        assert pos.shape == (n, 3)
        x = torch.ones(n, 2, 32, requires_grad=True)
        for y in (ops.rotary_axes(x, pos, f, (4, 5, 7)), ops.qk_norm_rotary(x, None, None, pos, f, (4, 5, 7))):
            torch.autograd.grad(y, x, torch.ones_like(y))
        at = {'tmae_rotary_axes': 9, 'tmae_qk_norm_rotary_fwd': 14, 'tmae_qk_norm_rotary_bwd': 15}         # ldpos
        assert len(seen) == 4 and all(a[at[name]] >= 3 for name, a in seen), [(name, a[at[name]]) for name, a in seen]
        seen.clear()


@pytest.mark.gpu
def test_one_tokens_positions_transposed():
    from tmae_amd import ops
    f = ops.rotary_freqs((4, 5, 7), device='cuda')
    x = torch.randn(1, 2, 32, device='cuda')
    parts = [torch.tensor([t], dtype=torch.int32, device='cuda') for t in (3, 1, 4)]
    apart = torch.arange(9, device='cuda').view(1, 9)[:, ::4]
    for pos in (torch.stack(parts).t(), apart):
        plain = pos.clone(memory_format=torch.contiguous_format).reshape(-1).clone().view(1, 3)
        assert torch.equal(ops.rotary_axes(x, pos, f, (4, 5, 7)), ops.rotary_axes(x, plain, f, (4, 5, 7)))
        assert torch.equal(ops.qk_norm_rotary(x, None, None, pos, f, (4, 5, 7)), ops.qk_norm_rotary(x, None, None, plain, f, (4, 5, 7)))


@pytest.mark.gpu
def test_angles_of_any_size():
    """Positions up to the ends of their types: the pair (1, 0) turns into the cosine and sine of the float64 product.  Their error is that
    of any angle (2 u); infinities and NaN have no angle."""
    import math
    from tmae_amd import ops
    g = torch.Generator().manual_seed(12)
    sections = (3, 2)
    f = ops.rotary_freqs(sections, 100.0)
    f[4] = 3e5                                                                          # (the frequencies are the caller's)
    big = torch.randint(-(1 << 62), 1 << 62, (400, 2), generator=g)
    stamps = 1_700_000_000_000_000_000 + torch.randint(0, 1 << 50, (400, 2), generator=g)
    ends = torch.tensor([[(1 << 63) - 1, -(1 << 63)], [1 << 53, (1 << 53) + 2], [0, 1], [(1 << 45) - 1, 1 << 45], [-(1 << 45), 1 << 46]])
    ladder = torch.tensor([[1 << s, -(1 << s) - 1] for s in range(63)])
    sizes = torch.rand(900, 2, generator=g) * 38
    floats = (10.0 ** sizes).float() * (torch.randint(0, 2, (900, 2), generator=g) * 2 - 1)
    edges = torch.tensor([[3.4028234e38, -3.4028234e38], [1e-30, 0.0], [2.0 ** 45, 2.0 ** 44], [1e30, 1.765e18]])
    for pos in (torch.cat([big, stamps, ends, ladder]), torch.cat([floats, edges])):
        n = pos.shape[0]
        theta = (pos.double()[:, [0, 0, 0, 1, 1]] * f[None]).tolist()
        want = torch.tensor([[[math.cos(t), math.sin(t)] for t in row] for row in theta], dtype=torch.float64)
        for interleaved in (False, True):
            x = torch.zeros(n, 1, 10)
            x[..., 0::2 if interleaved else 1][..., :5] = 1.0
            y = ops.rotary_axes(x.cuda(), pos.cuda(), f.cuda(), sections, interleaved=interleaved).cpu()[:, 0].double()
            got = torch.stack([y[:, 0::2], y[:, 1::2]], -1) if interleaved else torch.stack([y[:, :5], y[:, 5:]], -1)
            assert (got.abs() <= 1 + 2 * U).all()
            assert ((got - want).abs() <= 2 * U).all(), float((got - want).abs().max() / U)
    pos = torch.tensor([[float('inf'), 1.0], [1.0, -float('inf')], [float('nan'), 1.0], [1.0, 1.0]])
    y = ops.rotary_axes(torch.ones(4, 1, 10, device='cuda'), pos.cuda(), f.cuda(), sections, interleaved=True).cpu()[:, 0]
    assert torch.equal(y.isnan(), torch.tensor([[True] * 6 + [False] * 4, [False] * 6 + [True] * 4, [True] * 6 + [False] * 4, [False] * 10]))
