"""Scaled-dot-product attention inside 8x8 windows (ops.win_attn_dot) against the definition in 64 bits, and the chain
q/k norms + rotation -> attention as an encoder layer runs it.

Tolerances (u = 2^-24, e = eps / 2 of the stored type, bf16 2^-8; T = 64 tokens of a window at most).  Per query, A = the largest
scale * sum |q_c k_c| of its keys:
 * a logit is off by (dh + 4) u A; the exponent's argument and the sum's reciprocal round once more each (of a size up to A + 6): a
   probability is off by rho = 2 (dh + 8) u (A + 6) + (T + 16) u of itself, and by e more where it is rounded to the type for a product;
 * out: (rho + e + 4 T u) sum_j P |v| + e |out|;          dv: the same with sum_i P |dO|;
 * dS = scale P (dP - D), with G = sum |dO v| per pair and Dm = sum_j P G: off by
   eta = (2 rho + (dh + T + 8) u + e) scale P (G + Dm);    dq: sum_j (eta + T u |dS|) |k| + e |dq|;    dk: sum_i of the same with |q|."""
import ctypes

import pytest
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2 if dtype == torch.bfloat16 else 0.0


def within(got, want, tol, what):
    got = got.detach().double().cpu()
    assert torch.isfinite(want).all() and torch.isfinite(got).all(), what
    bad = ~((got - want).abs() <= tol + 1e-37)
    assert not bad.any(), f'{what}: {int(bad.sum())} of {bad.numel()}, worst {((got - want).abs() / tol.clamp_min(1e-300)).max():.3g} of the tolerance'


def place(counts, batch, ny, nx, g, shuffle=False):
    """counts: occupied cells of every frame -> the grid (-1: empty), and each row's (frame, y, x)"""
    grid = torch.full((batch, ny * nx), -1, dtype=torch.int32)
    cells = [torch.randperm(ny * nx, generator=g)[:c].sort().values for c in counts]
    flat = torch.cat([c + b * ny * nx for b, c in enumerate(cells)])
    rows = torch.randperm(flat.numel(), generator=g) if shuffle else torch.arange(flat.numel())
    grid.view(-1)[flat] = rows.int()
    at = torch.empty_like(flat)
    at[rows] = flat
    return grid.view(-1), torch.stack([at // (ny * nx), at % (ny * nx) // nx, at % nx], 1)


def window_of(at, shift):
    s = 4 if shift else 8
    return at[:, 0] * 10 ** 8 + (at[:, 1] + s) // 8 * 10 ** 4 + (at[:, 2] + s) // 8


def reference(q, k, v, do, same, nhead, scale):
    """[tokens, d] float64 and the mask of pairs that share a window -> results and tolerances without the rounding of the type"""
    if not q.shape[0] or not k.shape[0]:                                               # nothing attends to anything
        zeros = [torch.zeros_like(t) for t in (q, q, k, v)]
        return zeros, lambda e: zeros
    split = lambda t: t.view(t.shape[0], nhead, -1).transpose(0, 1)                    # noqa: E731
    join = lambda t: t.transpose(0, 1).reshape(t.shape[1], -1)                         # noqa: E731
    q, k, v, do = split(q), split(k), split(v), split(do)
    dh = q.shape[-1]
    logits = (q @ k.transpose(1, 2) * scale).masked_fill(~same, -float('inf'))
    top = logits.amax(-1, keepdim=True).clamp_min(-1e300)
    p = (logits - top).exp()
    total = p.sum(-1, keepdim=True)
    p = p / total.clamp_min(1e-300) * (total > 0)
    dp = do @ v.transpose(1, 2)
    ds = scale * p * (dp - (p * dp).sum(-1, keepdim=True))
    out = [join(t) for t in (p @ v, ds @ k, ds.transpose(1, 2) @ q, p.transpose(1, 2) @ do)]
    A = (q.abs() @ k.abs().transpose(1, 2) * scale).masked_fill(~same, 0).amax(-1, keepdim=True)

    def tolerances(e):
        T = 64
        rho = 2 * (dh + 8) * U * (A + 6) + (T + 16) * U
        gsum = (do.abs() @ v.abs().transpose(1, 2)) * same
        eta = (2 * rho + (dh + T + 8) * U + e) * scale * p * (gsum + (p * gsum).sum(-1, keepdim=True)) + T * U * ds.abs()
        wp = p * (rho + e + 4 * T * U)
        tols = [join(t) for t in (wp @ v.abs(), eta @ k.abs(), eta.transpose(1, 2) @ q.abs(), wp.transpose(1, 2) @ do.abs())]
        return [t + (e + 2 * U) * o.abs() for t, o in zip(tols, out)]
    return out, tolerances


CASES = [  # name, batch, ny, nx, queries, keys (None: self), heads, dh, shift, dtype, layout, work list, scale
    ('one_token', 1, 3, 5, [1], None, 1, 16, False, 'bf16', 'qkv', True, None),
    ('one_token_f32', 1, 1, 1, [1], None, 3, 64, True, 'f32', 'qk_v', False, None),
    ('full_window', 1, 8, 8, [64], None, 2, 32, False, 'bf16', 'qk_v', True, None),
    ('full_windows_shifted', 2, 24, 17, [408, 408], None, 4, 16, True, 'bf16', 'qkv', True, None),
    ('full_windows_64', 1, 16, 16, [256], None, 5, 64, False, 'bf16', 'qk_v', True, None),
    ('full_windows_f32', 1, 19, 21, [399], None, 3, 32, True, 'f32', 'qk_v', True, None),
    ('full_windows_f32_64', 1, 16, 16, [256], None, 1, 64, False, 'f32', 'qkv', True, None),
    ('sparse', 2, 70, 45, [160, 31], None, 8, 16, False, 'bf16', 'qk_v', True, None),
    ('sparse_dense_launch', 2, 70, 45, [160, 31], None, 8, 16, True, 'bf16', 'qk_v', False, None),
    ('ragged', 3, 40, 41, [900, 0, 333], None, 8, 32, True, 'bf16', 'qk_v', True, 0.4),
    ('ragged_f32', 2, 40, 41, [900, 333], None, 8, 16, False, 'f32', 'qkv', True, 0.03),
    ('seven_heads', 1, 33, 50, [700], None, 7, 16, True, 'bf16', 'qkv', True, None),
    ('cross', 2, 40, 41, [120, 300], [800, 13], 8, 32, True, 'bf16', 'q_k_v', True, None),
    ('cross_packed', 2, 40, 41, [120, 300], [800, 13], 8, 16, False, 'bf16', 'q_kv', True, None),
    ('cross_64', 1, 40, 41, [1100], [700], 2, 64, False, 'bf16', 'q_k_v', True, None),
    ('cross_f32', 2, 40, 41, [50, 900], [1600, 20], 5, 32, False, 'f32', 'q_kv', True, None),
    ('cross_dense_launch', 2, 40, 41, [50, 900], [1600, 20], 4, 16, True, 'bf16', 'q_k_v', False, None),
    ('cross_no_keys', 1, 20, 20, [90], [0], 4, 16, False, 'bf16', 'q_k_v', True, None),
    ('cross_no_queries', 1, 20, 20, [0], [90], 4, 16, False, 'f32', 'q_k_v', True, None),
    ('large_logits', 1, 30, 30, [600], None, 4, 32, False, 'bf16', 'qk_v', True, 9.0),
]


def make(case):
    name, batch, ny, nx, nq, nk, heads, dh, shift, dtype, layout, wl, scale = case
    g = torch.Generator().manual_seed(len(name) * 7 + ny)
    dt = {'bf16': torch.bfloat16, 'f32': torch.float32}[dtype]
    d = heads * dh
    grid_q, at_q = place(nq, batch, ny, nx, g, shuffle=True)
    grid_k, at_k = (grid_q, at_q) if nk is None else place(nk, batch, ny, nx, g)
    mq, mk = at_q.shape[0], at_k.shape[0]
    q, do = (torch.randn(mq, d, generator=g).to(dt) for _ in range(2))
    k, v = (torch.randn(mk, d, generator=g).to(dt) for _ in range(2))
    same = window_of(at_q, shift)[:, None] == window_of(at_k, shift)[None]
    return q, k, v, do, grid_q, grid_k, same


def pack(layout, q, k, v):
    return {'qkv': lambda: (torch.cat([q, k, v], 1), None, None), 'qk_v': lambda: (torch.cat([q, k], 1), v, None),
            'q_k_v': lambda: (q, k, v), 'q_kv': lambda: (q, torch.cat([k, v], 1), 'kv')}[layout]()


def unpack(layout, grads, d):
    if layout == 'qkv':
        return grads[0].split(d, 1)
    if layout == 'qk_v':
        return (*grads[0].split(d, 1), grads[1])
    return grads if layout == 'q_k_v' else (grads[0], *grads[1].split(d, 1))


# --------------------------------------------------------------------------------------------------------------- the CPU

def test_refusals():
    from tmae_amd import ops
    grid = torch.full((2 * 9 * 9,), -1, dtype=torch.int32)
    x, v = torch.zeros(10, 64), torch.zeros(10, 32)

    def call(a=x, b=v, c=None, gq=grid, gk=grid, nhead=2, batch=2, ny=9, nx=9, **k):
        return ops.win_attn_dot(a, b, c, gq, gk, nhead, batch, ny, nx, False, **k)
    with pytest.raises(RuntimeError, match='GPU only'):
        call()
    for kind, match, bad in (
            (ValueError, r'q\|k', dict(b=None, c=v)), (ValueError, 'kv', dict(c='vk')), (ValueError, 'one type', dict(b=v.bfloat16())),
            (TypeError, 'float32 / bfloat16', dict(a=x.half(), b=v.half())), (ValueError, 'rows of', dict(b=v[:, :16])),
            (ValueError, 'rows of', dict(b=v[:9])), (ValueError, 'rows of', dict(a=v, b=v, c=v[:3])), (ValueError, '16, 32 or 64', dict(nhead=4)),
            (ValueError, '16, 32 or 64', dict(nhead=0)), (ValueError, 'scale', dict(scale=0.0)), (ValueError, 'scale', dict(scale=-1.0)),
            (ValueError, 'scale', dict(scale=float('nan'))), (ValueError, 'scale', dict(scale=float('inf'))), (ValueError, 'grid', dict(batch=0)),
            (ValueError, 'grid_q', dict(gq=grid[:-1])), (ValueError, 'grid_k', dict(gk=grid.long())), (ValueError, 'grid_q', dict(nx=8)),
            (ValueError, 'work list', dict(worklist=torch.zeros(5, dtype=torch.int32)))):
        with pytest.raises(kind, match=match):
            call(**bad)


def test_c_entries_refuse_bad_arguments():
    from tmae_amd._lib import lib
    one = ctypes.c_void_p(16)

    def fwd(q=one, ldq=64, k=one, v=one, dtype=1, mq=4, mk=4, nhead=4, dh=16, gq=one, gk=one, batch=1, ny=8, nx=8, scale=1.0, out=one, ldo=64, wl=None):
        return lib.tmae_win_attn_dot_fwd(q, ldq, k, 64, v, 64, dtype, mq, mk, nhead, dh, gq, gk, batch, ny, nx, 0, scale, out, ldo, wl, None)
    assert fwd(mq=0) == 0 and fwd(dtype=3) == -3
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(gq=None), dict(gk=None), dict(mq=-1), dict(mk=-1),
                dict(mq=1 << 31), dict(nhead=0), dict(nhead=4097), dict(dh=8), dict(dh=48), dict(batch=0), dict(ny=0), dict(nx=0), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=float('nan')), dict(scale=float('inf')), dict(ldq=63), dict(ldq=56), dict(ldo=68 + 2),
                dict(q=ctypes.c_void_p(8)), dict(batch=1 << 20, ny=1 << 10, nx=1 << 10), dict(wl=one, ny=2041)):
        assert fwd(**bad) == -1, bad

    def bwd(dq=one, dk=one, dv=one, do=one, lddq=64):
        return lib.tmae_win_attn_dot_bwd(one, 64, one, 64, one, 64, do, 64, 1, 4, 4, 4, 16, one, one, 1, 8, 8, 0, 1.0, dq, lddq, dk, 64, dv,
                                         64, None, None)
    for bad in (dict(dq=None), dict(dk=None), dict(dv=None), dict(do=None), dict(lddq=60)):
        assert bwd(**bad) == -1, bad


# --------------------------------------------------------------------------------------------------------------- the GPU

@pytest.mark.gpu
@pytest.mark.parametrize('case', CASES, ids=lambda c: c[0])
def test_attention_and_its_gradients(case):
    from tmae_amd import ops
    name, batch, ny, nx, nq, nk, heads, dh, shift, dtype, layout, wl, scale = case
    q, k, v, do, grid_q, grid_k, same = make(case)
    d, e = heads * dh, half_step(q.dtype)
    want, tolerances = reference(q.double(), k.double(), v.double(), do.double(), same, heads, scale or dh ** -0.5)
    gq = grid_q.cuda()
    gk = gq if nk is None else grid_k.cuda()
    args = [t.cuda().requires_grad_() if torch.is_tensor(t) else t for t in pack(layout, q, k, v)]
    worklist = ops.window_worklist(gq, gk, batch, ny, nx, shift) if wl else None
    for covered in (True, False):
        o = ops.win_attn_dot(*args, gq, gk, heads, batch, ny, nx, shift, scale=scale, worklist=worklist, covered=covered)
        grads = torch.autograd.grad(o, [t for t in args if torch.is_tensor(t)], do.cuda())
        for what, got, w, t in zip(('out', 'dq', 'dk', 'dv'), (o, *unpack(layout, grads, d)), want, tolerances(e)):
            assert got.dtype == q.dtype
            within(got, w, t, f'{name} {what}')
        with torch.no_grad():
            assert torch.equal(ops.win_attn_dot(*args, gq, gk, heads, batch, ny, nx, shift, scale=scale, worklist=worklist, covered=covered), o)


@pytest.mark.gpu
def test_gradient_against_differences():
    """The float32 gradients along a direction against differences of the 64-bit definition."""
    from tmae_amd import ops
    case = ('differences', 2, 40, 41, [120, 300], [800, 13], 4, 16, True, 'f32', 'q_k_v', True, None)
    q, k, v, do, grid_q, grid_k, same = make(case)
    g = torch.Generator().manual_seed(5)
    ways = [torch.randn(t.shape, generator=g).double() for t in (q, k, v)]
    h = 1e-6
    hi, lo = ((reference(*(t.double() + s * h * w for t, w in zip((q, k, v), ways)), do.double(), same, 4, 0.25)[0][0] * do.double()).sum()
              for s in (1, -1))
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    gq, gk = grid_q.cuda(), grid_k.cuda()
    o = ops.win_attn_dot(*leaves, gq, gk, 4, 2, 40, 41, True, worklist=ops.window_worklist(gq, gk, 2, 40, 41, True))
    grads = torch.autograd.grad(o, leaves, do.cuda())
    along = sum((gr.double().cpu() * w).sum() for gr, w in zip(grads, ways))
    size = sum((gr.double().cpu() * w).abs().sum() for gr, w in zip(grads, ways))
    assert abs((hi - lo) / (2 * h) - along) <= 1e-5 * size


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_rows_outside_the_grids(dtype):
    """Rows that stand in no cell (dropped tokens) stay zero, entries that are no row count as empty cells, with and without a list."""
    from tmae_amd import ops
    g = torch.Generator().manual_seed(2)
    grid, at = place([300], 1, 24, 24, g)
    q, k, v, do = (torch.randn(300, 64, generator=g).to(dtype) for _ in range(4))
    gone = torch.randperm(300, generator=g)[:80]
    kept = torch.ones(300, dtype=torch.bool)
    kept[gone] = False
    masked = torch.where(grid >= 0, torch.where(kept[grid.clamp(min=0).long()], grid, torch.full_like(grid, -1)), grid)
    odd = torch.where((grid >= 0) & (masked < 0), torch.full_like(grid, 300) + (torch.arange(grid.numel()) % 2) * 2 ** 30, masked).int()
    same = (window_of(at, False)[:, None] == window_of(at, False)[None]) & kept[:, None] & kept[None]
    want, tolerances = reference(q.double(), k.double(), v.double(), do.double(), same, 4, 0.25)
    for gr in (masked, odd):
        for other in (False, True):
            gq = gr.cuda()
            gk = gr.cuda() if other else gq
            for worklist in (None, ops.window_worklist(masked.cuda(), masked.cuda(), 1, 24, 24, False)):
                leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
                o = ops.win_attn_dot(*leaves, gq, gk, 4, 1, 24, 24, False, worklist=worklist)
                grads = torch.autograd.grad(o, leaves, do.cuda())
                for what, got, w, t in zip(('out', 'dq', 'dk', 'dv'), (o, *grads), want, tolerances(half_step(dtype))):
                    within(got, w, t, what)
                    assert not got[gone.cuda()].any()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('value', [float('nan'), float('inf'), -float('inf')])
def test_a_bad_token_stays_in_its_window_and_head(dtype, value):
    """What a NaN or an infinity reaches ends at its window and head, in every output, whichever tensor holds it."""
    from tmae_amd import ops
    g = torch.Generator().manual_seed(4)
    for counts, ny in (([60], 40), ([700], 40), ([1600], 40)):
        grid, at = place(counts, 1, ny, ny, g)
        n, h, dh = counts[0], 6, 16
        gr = grid.cuda()
        wl = ops.window_worklist(gr, gr, 1, ny, ny, True)
        win = window_of(at, True)
        for which in range(4):
            tensors = [torch.randn(n, h * dh, generator=g) for _ in range(4)]
            tensors[which][n // 2, 2 * dh + 3] = value
            q, k, v, do = (t.to(dtype).cuda() for t in tensors)
            leaves = [t.requires_grad_() for t in (q, k, v)]
            o = ops.win_attn_dot(*leaves, gr, gr, h, 1, ny, ny, True, worklist=wl, covered=True)
            for t in (o, *torch.autograd.grad(o, leaves, do)):
                fine = torch.isfinite(t.detach().float().view(n, h, dh)).all(-1).cpu()
                touched = torch.zeros(n, h, dtype=torch.bool)
                touched[win == win[n // 2], 2] = True
                assert fine[~touched].all()
            # (a key's infinity gives a logit of -inf where the query's channel has the other sign: probability 0, and all is finite)
            assert which == 3 or value == value or not torch.isfinite(o[n // 2]).all()


@pytest.mark.gpu
def test_norms_rotation_and_attention_together():
    """As an encoder layer uses them: one packed projection, norms and rotation, attention, all gradients -- against autograd through
    the definition in 64 bits; the same bits again on another stream and from a captured graph on new inputs."""
    from tmae_amd import ops
    g = torch.Generator().manual_seed(9)
    batch, ny, nx, h, dh, sec = 2, 40, 41, 8, 16, (2, 3, 3)
    grid, at = place([500, 301], batch, ny, nx, g)
    n, d = at.shape[0], h * dh
    same = window_of(at, True)[:, None] == window_of(at, True)[None]
    pos = torch.cat([torch.zeros(n, 1, dtype=torch.int64), at[:, 1:]], 1).int()
    f = ops.rotary_freqs(sec, 100.0)
    gq, gk = (1 + 0.2 * torch.randn(dh, generator=g) for _ in range(2))
    qk, v, do = (torch.randn(n, w, generator=g) for w in (2 * d, d, d))

    def definition(qk, gq, gk, v):
        x = qk.view(n, 2 * h, dh)
        x = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        x = torch.cat([x[:, :h] * gq, x[:, h:] * gk], 1)
        theta = (pos.double()[:, torch.repeat_interleave(torch.arange(3), torch.tensor(sec))] * f)[:, None]
        a, b = x[..., :8], x[..., 8:]
        x = torch.cat([a * theta.cos() - b * theta.sin(), a * theta.sin() + b * theta.cos()], -1)
        q, k = x[:, :h].transpose(0, 1), x[:, h:].transpose(0, 1)
        p = torch.softmax((q @ k.transpose(1, 2) * dh ** -0.5).masked_fill(~same, -float('inf')), -1)
        return (p @ v.view(n, h, dh).transpose(0, 1)).transpose(0, 1).reshape(n, d)

    gr, posg, fg = grid.cuda(), pos.cuda(), f.cuda()
    wl = ops.window_worklist(gr, gr, batch, ny, nx, True)

    def run(qk, gq, gk, v, do):
        y = ops.qk_norm_rotary(qk.view(n, 2 * h, dh), gq, gk, posg, fg, sec)
        o = ops.win_attn_dot(y.view(n, 2 * d), v, None, gr, gr, h, batch, ny, nx, True, worklist=wl, covered=True)
        return (o.detach(), *torch.autograd.grad(o, (qk, gq, gk, v), do))

    # bf16: the rows between the two operators are rounded once more each way (2^-8 of a unit-size row, through logits of size ~ 4 and
    # sums of mixed signs: 2-norms within 4 roundings); float32: every step within a few hundred u
    for dtype, bound in ((torch.float32, 400 * U), (torch.bfloat16, 4 * 2.0 ** -8)):
        rounded = [t.to(dtype) for t in (qk, v, do)]
        ref_in = [rounded[0].double().requires_grad_(), gq.double().requires_grad_(), gk.double().requires_grad_(), rounded[1].double().requires_grad_()]
        ref = definition(*ref_in)
        want = (ref.detach(), *torch.autograd.grad(ref, ref_in, rounded[2].double()))
        gpu = [rounded[0].cuda().requires_grad_(), gq.cuda().requires_grad_(), gk.cuda().requires_grad_(), rounded[1].cuda().requires_grad_()]
        got = run(*gpu, rounded[2].cuda())
        for i, (a, b) in enumerate(zip(got, want)):
            assert (a.double().cpu() - b).norm() <= bound * b.norm(), (dtype, i, float((a.double().cpu() - b).norm() / b.norm()))
    # another stream, then a graph replayed on new inputs with eager work between
    dog = do.bfloat16().cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run(*gpu, dog)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(again, got))
    held = [t.detach().clone().requires_grad_() for t in gpu]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*held, dog)
    for k in range(4):
        fresh = [torch.randn(t.shape, generator=g).to(t.dtype).cuda().requires_grad_() for t in gpu]
        with torch.no_grad():
            for a, b in zip(held, fresh):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, run(*fresh, dog))), k


# ------------------------------------------------------------------------------------------------ the layers that call them

OPTIONS = [{'cosine': False}, {'cosine': True, 'tau_min': 0.01, 'rotary': {'SECTIONS': [4, 4]}},
           {'cosine': False, 'rotary': {'SECTIONS': [2, 3, 3], 'BASE': 50.0}},
           {'cosine': False, 'rotary': {'SECTIONS': [2, 3, 3], 'BASE': 50.0}, 'qk_norm': True}]


def test_options_build_and_train_their_gains():
    from tmae_amd.modules.sst import WindowAttention, WindowCrossAttention
    from tmae_amd.train.optim import reference_param_groups
    for opt in OPTIONS:
        m = WindowAttention(128, 8, 0.0, opt).self_attn
        names = set(dict(m.named_parameters()))
        assert ('tau' in names) == opt['cosine'] and ('q_norm.weight' in names) == bool(opt.get('qk_norm'))
        if opt.get('qk_norm'):
            plain, _, rest = reference_param_groups(m)
            assert any(p is m.q_norm.weight for p in plain) and any(p is m.k_norm.weight for p in plain)
    for bad, kind in (({'cosine': False, 'qk_norm': True}, NotImplementedError), ({'rotary': {'SECTIONS': [8]}}, ValueError),
                      ({'rotary': {'SECTIONS': [4, 5]}}, ValueError), ({'rotary': {'SECTIONS': [0, 5]}}, ValueError)):
        with pytest.raises(kind):
            WindowCrossAttention(128, 8, 0.0, bad)


def layer_reference(a, W, b, x, x_kv, at_q, at_k, tq, tk, table, shift, opt, tau):
    """q, k, v from the packed in-projection -> attention rows before the out-projection, float64"""
    d, h, dh = 128, 8, 16
    s = 4 if shift else 8
    cell = lambda at: (at[:, 1] + s) % 8 * 8 + (at[:, 2] + s) % 8                      # noqa: E731
    rot = opt.get('rotary')
    q_in, k_in = (x, x_kv) if rot else (x + table[cell(at_q)], x_kv + table[cell(at_k)])
    q = (q_in @ W[:d].t() + b[:d]).view(-1, h, dh)
    k = (k_in @ W[d:2 * d].t() + b[d:2 * d]).view(-1, h, dh)
    v = (x_kv @ W[2 * d:].t() + b[2 * d:]).view(-1, h, dh)
    if opt.get('qk_norm'):
        q = q * (q.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * a['q_norm.weight']
        k = k * (k.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * a['k_norm.weight']
    if rot:
        sec = rot['SECTIONS']
        axis = torch.repeat_interleave(torch.arange(len(sec)), torch.tensor(sec))
        f = torch.cat([torch.tensor(float(rot.get('BASE', 100.0)), dtype=torch.float64) ** (-torch.arange(p).double() / p) for p in sec])

        def turned(t, at, time):
            pos = at.clone().double()
            pos[:, 0] = time
            th = (pos[:, 3 - len(sec):][:, axis] * f)[:, None]
            p = th.shape[-1]
            lo, hi = t[..., :p], t[..., p:2 * p]
            return torch.cat([lo * th.cos() - hi * th.sin(), lo * th.sin() + hi * th.cos(), t[..., 2 * p:]], -1)
        q, k = turned(q, at_q, tq), turned(k, at_k, tk)
    scale = dh ** -0.5
    if opt['cosine']:
        q, k, scale = q / q.norm(dim=-1, keepdim=True), k / k.norm(dim=-1, keepdim=True), 1.0 / a['tau'].view(())
    same = window_of(at_q, shift)[:, None] == window_of(at_k, shift)[None]
    logits = (q.transpose(0, 1) @ k.permute(1, 2, 0) * scale).masked_fill(~same, -1e30)
    p = torch.softmax(logits, -1) * same
    return (p @ v.transpose(0, 1)).transpose(0, 1).reshape(-1, d)


@pytest.mark.gpu
@pytest.mark.parametrize('cross', [False, True])
@pytest.mark.parametrize('opt', OPTIONS, ids=['dot', 'cosine_rotary', 'dot_rotary', 'dot_rotary_norm'])
def test_layers_with_the_options(opt, cross):
    """Self and cross attention layers in float32, outputs and every gradient against autograd through the definition in 64 bits.
    2-norms: projections over 128 channels (128 u each way), norms, rotation and attention (400 u, above), the weight gradients' sums
    over 800 rows (800 u) -- within 1500 u together."""
    from tmae_amd.modules.sparse import SparseConvTensor
    from tmae_amd.modules.sst import WindowAttention, WindowCrossAttention, WindowPlan, pos_embed_table
    g = torch.Generator().manual_seed(21)
    ny, nx = 40, 41
    (_, at_q), (_, at_k) = place([500, 300], 2, ny, nx, g), place([90, 700], 2, ny, nx, g)
    table = pos_embed_table(128, [8, 8, 1], 1000)
    x, x_kv = (torch.randn(t.shape[0], 128, generator=g) for t in (at_q, at_k))
    do = torch.randn(800, 128, generator=g)
    torch.manual_seed(3)
    layer = (WindowCrossAttention if cross else WindowAttention)(128, 8, 0.0, opt)
    params = layer.cross_attn if cross else layer.self_attn
    with torch.no_grad():
        for n, t in params.named_parameters():
            if 'norm' in n or 'bias' in n:
                t.add_(0.2 * torch.randn(t.shape))
    names = [n for n, _ in params.named_parameters() if not (cross and n.startswith('out_proj'))]
    ref = {n: t.detach().double().requires_grad_() for n, t in params.named_parameters()}
    layer.cuda()
    for shift in (False, True):
        xr, kr = x.double().requires_grad_(), x_kv.double().requires_grad_()
        kv = kr if cross else xr
        o = layer_reference(ref, ref['in_proj_weight'], ref['in_proj_bias'], xr, kv, at_q, at_k if cross else at_q, 0, -1 if cross else 0,
                            table.double(), shift, opt, None)
        if not cross:
            o = o @ ref['out_proj.weight'].t() + ref['out_proj.bias']
        leaves = [xr] + ([kr] if cross else []) + [ref[n] for n in names]
        want = [o.detach(), *torch.autograd.grad(o, leaves, do.double())]
        xg, kg = x.cuda().requires_grad_(), x_kv.cuda().requires_grad_()
        plan_k = WindowPlan(SparseConvTensor(kg, at_k.int().cuda(), [ny, nx], 2))
        plan = WindowPlan(SparseConvTensor(xg, at_q.int().cuda(), [ny, nx], 2), other=plan_k if cross else None)
        args = (xg, plan, kg, plan_k) if cross else (xg, plan)
        og = layer(*args, table.cuda(), [8, 8, 1], shift)[0]
        got = [og.detach(), *torch.autograd.grad(og, [xg] + ([kg] if cross else []) + [dict(params.named_parameters())[n] for n in names],
                                                 do.cuda())]
        for n, a, b in zip(['out', 'dx'] + (['dx_kv'] if cross else []) + names, got, want):
            off = float((a.double().cpu() - b).norm())
            assert off <= 1500 * U * float(b.norm()) + 1e-6 * (n == 'tau'), (n, shift, off / float(b.norm()))


@pytest.mark.gpu
@pytest.mark.parametrize('amp', [False, True])
def test_model_step_with_the_options(amp):
    """A training step of the model built with the options: every parameter of the layers gets a finite gradient that is not zero."""
    from conftest import build_product_model
    from pcdet.models import model_fn_decorator

    def edit(c):
        for blk in c.MODEL.BACKBONE_3D.SST_BLOCK_LIST:
            pairs = blk.ENCODER.D_MODEL // blk.ENCODER.NHEAD // 2
            blk.ENCODER.LAYER_CFG = {'cosine': False, 'qk_norm': True, 'rotary': {'SECTIONS': [pairs // 4, pairs // 4, pairs // 2], 'BASE': 100.0}}
    torch.manual_seed(0)
    model, _, ds = build_product_model(2, device='cuda', n_points=6000, cfg_edit=edit)
    model.train()
    with torch.autocast('cuda', dtype=torch.bfloat16, enabled=amp):
        loss = model_fn_decorator()(model, ds.batch(0)).loss
    loss.backward()
    assert torch.isfinite(loss)
    seen = 0
    for n, p in model.named_parameters():
        if 'win_attn' in n:
            assert p.grad is not None and torch.isfinite(p.grad).all(), n
            seen += int('norm.weight' in n)
            # (a bias of all keys moves every logit of a query alike where no rotation stands between: not so here)
            assert p.grad.abs().max() > 0, n
    assert seen >= 16


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_an_infinite_value_stays_an_infinity(dtype):
    """v_j = inf in a channel: that channel of every query of the window is inf (all probabilities are above 0), the others are finite;
    dO_i = inf: the same of dV.  The bad token is the first of its window, which the slots behind the last one stand for."""
    from tmae_amd import ops
    g = torch.Generator().manual_seed(6)
    for dh, h in ((16, 5), (32, 2), (64, 2)):
        for count in (40, 300, 900, 1600):                                              # 1 to 64 tokens a window
            grid, at = place([count], 1, 40, 40, g)
            gr = grid.cuda()
            win = window_of(at, False)
            first = torch.stack([(win == w).nonzero()[0, 0] for w in win.unique()])
            touched = torch.zeros(count, h * dh, dtype=torch.bool)
            touched[:, dh + 3] = True
            q, k, v, do = (torch.randn(count, h * dh, generator=g).to(dtype) for _ in range(4))
            bad_v, bad_do = v.clone(), do.clone()
            bad_v[first, dh + 3] = float('inf')
            bad_do[first, dh + 3] = float('inf')
            for worklist in (None, ops.window_worklist(gr, gr, 1, 40, 40, False)):
                run = lambda v: ops.win_attn_dot(q.cuda(), k.cuda(), v, gr, gr, h, 1, 40, 40, False, worklist=worklist, covered=True)  # noqa: E731
                o = run(bad_v.cuda()).cpu().float()
                assert (o[touched] == float('inf')).all() and torch.isfinite(o[~touched]).all()
                leaf = v.cuda().requires_grad_()
                dv = torch.autograd.grad(run(leaf), leaf, bad_do.cuda())[0].cpu().float()
                assert (dv[touched] == float('inf')).all() and torch.isfinite(dv[~touched]).all()


@pytest.mark.gpu
def test_a_second_derivative_is_refused():
    from tmae_amd import ops
    grid = torch.arange(64, dtype=torch.int32, device='cuda')
    x = torch.randn(64, 48, device='cuda', requires_grad=True)
    o = ops.win_attn_dot(x, None, None, grid, grid, 1, 1, 8, 8, False)
    dx, = torch.autograd.grad(o.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match='once_differentiable'):
        (o.sum() + dx.sum()).backward()


@pytest.mark.gpu
def test_rows_beyond_32_bits():
    """2.25 M rows of 2048 bytes: the last frame's results are those of the last frame alone."""
    from tmae_amd import ops
    batch, ny, nx, h, dh = 9, 500, 500, 8, 64
    cells, d = ny * nx, h * dh
    g = torch.Generator(device='cuda').manual_seed(1)
    qk, v, do = (torch.randn(batch * cells, w, generator=g, device='cuda', dtype=torch.bfloat16) for w in (2 * d, d, d))
    assert qk.numel() * 2 > 2 ** 32
    grid = torch.arange(batch * cells, dtype=torch.int32, device='cuda')

    def run(qk, v, do, grid, batch):
        leaves = [t.detach().requires_grad_() for t in (qk, v)]
        o = ops.win_attn_dot(*leaves, None, grid, grid, h, batch, ny, nx, True, covered=True,
                             worklist=ops.window_worklist(grid, grid, batch, ny, nx, True))
        return [t.detach() for t in (o, *torch.autograd.grad(o, leaves, do))]
    whole = run(qk, v, do, grid, batch)
    alone = run(qk[-cells:], v[-cells:], do[-cells:], grid[:cells], 1)
    for a, b in zip(whole, alone):
        assert torch.equal(a[-cells:], b)


@pytest.mark.gpu
@pytest.mark.parametrize('worklist', [True, False])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('heads,dh,shift,cross', [(8, 16, False, False), (3, 16, True, True), (4, 32, True, False), (3, 32, False, True),
                                                  (2, 64, False, False), (1, 64, True, True)])
def test_many_frames(heads, dh, shift, cross, dtype, worklist):
    """More tokens than the variants for few of them take, of every size of window: the first and the last frame against the definition."""
    from tmae_amd import ops
    g = torch.Generator().manual_seed(dh + heads)
    batch, ny, nx, d, e = 25, 40, 41, heads * dh, half_step(dtype)
    counts = [(60, 300, 700, 1300, 1640)[b % 5] for b in range(batch)]
    grid_q, at_q = place(counts, batch, ny, nx, g)
    grid_k, at_k = place(counts[::-1], batch, ny, nx, g) if cross else (grid_q, at_q)
    mq, mk = at_q.shape[0], at_k.shape[0]
    assert mq + mk > 32768
    q, do = (torch.randn(mq, d, generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(mk, d, generator=g).to(dtype) for _ in range(2))
    gq = grid_q.cuda()
    gk = grid_k.cuda() if cross else gq
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    wl = ops.window_worklist(gq, gk, batch, ny, nx, shift) if worklist else None
    o = ops.win_attn_dot(*leaves, gq, gk, heads, batch, ny, nx, shift, worklist=wl, covered=True)
    got = [o, *torch.autograd.grad(o, leaves, do.cuda())]
    for frame in (0, batch - 1):
        fq, fk = at_q[:, 0] == frame, at_k[:, 0] == frame
        same = window_of(at_q[fq], shift)[:, None] == window_of(at_k[fk], shift)[None]
        want, tolerances = reference(q[fq].double(), k[fk].double(), v[fk].double(), do[fq].double(), same, heads, dh ** -0.5)
        for what, t, rows, w, tol in zip(('out', 'dq', 'dk', 'dv'), got, (fq, fq, fk, fk), want, tolerances(e)):
            within(t[rows.cuda()], w, tol, f'{what} of frame {frame}')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_rows_from_any_address(dtype):
    """Pieces of flat buffers that begin beside a 16-byte boundary, rows apart and a broadcast gradient: the same bits as aligned ones."""
    from tmae_amd import ops
    g = torch.Generator(device='cuda').manual_seed(8)
    grid = torch.arange(24 * 24, dtype=torch.int32, device='cuda')
    qk, v, row = (torch.randn(n, generator=g, device='cuda').to(dtype) for n in (576 * 64, 576 * 32, 32))

    def run(qk, v, do):
        leaves = [t.detach().requires_grad_() for t in (qk, v)]
        o = ops.win_attn_dot(*leaves, None, grid, grid, 2, 1, 24, 24, True, covered=True)
        return [t.detach() for t in (o, *torch.autograd.grad(o, leaves, do))]

    def beside(t):
        flat = torch.zeros(t.numel() + 1, device='cuda', dtype=dtype)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)
    qk, v, do = qk.view(576, 64), v.view(576, 32), row.expand(576, 32)
    want = run(qk, v, do.contiguous())
    wide = torch.zeros(576, 100, device='cuda', dtype=dtype)
    wide[:, 3:67] = qk
    for args in ((beside(qk), beside(v), beside(do)), (wide[:, 3:67], v, do)):
        for a, b in zip(run(*args), want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_large_calls_in_a_graph_and_side_by_side():
    """Norms, rotation and attention over more tokens than the variants for few of them take: replays on new inputs, with eager work
    between them, and calls at once on two streams give the bits of a call alone."""
    from tmae_amd import ops
    g = torch.Generator(device='cuda').manual_seed(3)
    batch, ny, nx, h, dh, sec = 4, 100, 99, 8, 16, (2, 3, 3)
    n, d = batch * ny * nx, h * dh
    grid = torch.arange(n, dtype=torch.int32, device='cuda')
    wl = ops.window_worklist(grid, grid, batch, ny, nx, True)
    pos = torch.randint(0, 99, (n, 3), generator=g, device='cuda', dtype=torch.int32)
    f = ops.rotary_freqs(sec, 100.0, 'cuda')

    def inputs():
        return [torch.randn(s, generator=g, device='cuda').to(t) for s, t in (((n, 2 * d), torch.bfloat16), ((n, d), torch.bfloat16),
                                                                              ((dh,), torch.float32), ((dh,), torch.float32))]

    def run(qk, v, gq, gk, do):
        leaves = [t.detach().requires_grad_() for t in (qk, v, gq, gk)]
        turned = ops.qk_norm_rotary(leaves[0].view(n, 2 * h, dh), *leaves[2:], pos, f, sec).view(n, 2 * d)
        o = ops.win_attn_dot(turned, leaves[1], None, grid, grid, h, batch, ny, nx, True, worklist=wl, covered=True)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]
    do = torch.randn(n, d, generator=g, device='cuda').bfloat16()
    held = inputs()
    run(*held, do)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*held, do)
    for k in range(3):
        fresh = inputs()
        for a, b in zip(held, fresh):
            a.copy_(b)
        graph.replay()
        want = run(*fresh, do)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k
    sets = [inputs() for _ in range(2)]
    alone = [run(*s, do) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        both = []
        for stream, s in zip(streams, sets):
            with torch.cuda.stream(stream):
                both.append(run(*s, do))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(both, alone) for a, b in zip(x, y))


@pytest.mark.gpu
@pytest.mark.parametrize('heads,dh', [(4, 16), (2, 32), (1, 64)])
def test_infinities_in_large_calls(heads, dh):
    """As in small ones: an infinite dO of a window's first token makes that channel of dV infinite in its window, and nothing else."""
    from tmae_amd import ops
    g = torch.Generator().manual_seed(dh)
    batch, ny, nx = 12, 40, 41
    grid, at = place([(60, 300, 700, 1300, 1640)[b % 5] for b in range(batch)], batch, ny, nx, g)
    n = at.shape[0]
    assert 2 * n > 8192
    win = window_of(at, False)
    order = torch.argsort(win, stable=True)
    first = order[torch.cat([torch.ones(1, dtype=torch.bool), win[order][1:] != win[order][:-1]])]
    touched = torch.zeros(n, heads * dh, dtype=torch.bool)
    touched[:, 5] = True
    q, k, v, do = (torch.randn(n, heads * dh, generator=g).bfloat16() for _ in range(4))
    do[first, 5] = float('inf')
    gr = grid.cuda()
    for worklist in (None, ops.window_worklist(gr, gr, batch, ny, nx, False)):
        leaf = v.cuda().requires_grad_()
        o = ops.win_attn_dot(q.cuda(), k.cuda(), leaf, gr, gr, heads, batch, ny, nx, False, worklist=worklist, covered=True)
        dv = torch.autograd.grad(o, leaf, do.cuda())[0].cpu().float()
        assert torch.isfinite(o).all() and (dv[touched] == float('inf')).all() and torch.isfinite(dv[~touched]).all()


TWO_PARTS = 2.0 ** -15         # a probability as two bfloat16: cut to 8 bits (the rest is below 2^-7 of it), the rest rounded (2^-8 of that)


def two_parts(p):
    high = (p.float().view(torch.int32) & -65536).view(torch.float32)
    return high.double() + (p.float() - high).bfloat16().double()


def test_the_tolerance_tells_one_rounding_of_the_probabilities_from_two_parts():
    """The bound of the next test holds for P and dS as two bfloat16 and not for either of them rounded to one."""
    case = [c for c in CASES if c[0] == 'ragged'][0]
    q, k, v, do, _, _, same = (t.double() if t.is_floating_point() else t for t in make(case))
    h, scale = 8, 0.4
    want, tolerances = reference(q, k, v, do, same, h, scale)
    tols = [t + half_step(torch.bfloat16) * w.abs() for t, w in zip(tolerances(TWO_PARTS), want)]
    heads = lambda t: t.view(t.shape[0], h, -1).transpose(0, 1)                        # noqa: E731
    rows = lambda t: t.transpose(0, 1).reshape(t.shape[1], -1)                         # noqa: E731
    p = torch.softmax((heads(q) @ heads(k).transpose(1, 2) * scale).masked_fill(~same, -float('inf')), -1)
    dp = heads(do) @ heads(v).transpose(1, 2)
    ds = scale * p * (dp - (p * dp).sum(-1, keepdim=True))
    for part, fits in ((two_parts, True), (lambda t: t.bfloat16().double(), False)):
        results = (part(p) @ heads(v), part(ds) @ heads(k), part(ds).transpose(1, 2) @ heads(q), part(p).transpose(1, 2) @ heads(do))
        for got, w, tol in zip(results, want, tols):
            assert ((rows(got).bfloat16().double() - w).abs() <= tol).all() == fits


@pytest.mark.gpu
@pytest.mark.parametrize('worklist', [True, False])
@pytest.mark.parametrize('batch', [1, 9])
@pytest.mark.parametrize('heads,dh,shift,cross', [(8, 16, False, False), (3, 16, True, True), (4, 32, True, False), (3, 32, False, True),
                                                  (2, 64, False, False), (1, 64, True, True)])
def test_probabilities_and_their_gradients_keep_two_parts(heads, dh, shift, cross, batch, worklist):
    """bfloat16 results carry their own rounding and P and dS as two bfloat16, however many tokens the call has: the first and the last
    frame against the definition, with 2^-15 of a probability where `test_many_frames` allows a rounding of 2^-8."""
    from tmae_amd import ops
    g = torch.Generator().manual_seed(dh + heads + batch)
    ny, nx, d, e = 40, 41, heads * dh, half_step(torch.bfloat16)
    counts = [(1300, 300, 700, 60, 1640)[b % 5] for b in range(batch)]
    grid_q, at_q = place(counts, batch, ny, nx, g)
    grid_k, at_k = place(counts[::-1], batch, ny, nx, g) if cross else (grid_q, at_q)
    mq, mk = at_q.shape[0], at_k.shape[0]
    assert (mq + mk > 8192) == (batch > 1)
    q, do = (torch.randn(mq, d, generator=g).bfloat16() for _ in range(2))
    k, v = (torch.randn(mk, d, generator=g).bfloat16() for _ in range(2))
    gq = grid_q.cuda()
    gk = grid_k.cuda() if cross else gq
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    wl = ops.window_worklist(gq, gk, batch, ny, nx, shift) if worklist else None
    o = ops.win_attn_dot(*leaves, gq, gk, heads, batch, ny, nx, shift, worklist=wl, covered=True)
    got = [o, *torch.autograd.grad(o, leaves, do.cuda())]
    for frame in {0, batch - 1}:
        fq, fk = at_q[:, 0] == frame, at_k[:, 0] == frame
        same = window_of(at_q[fq], shift)[:, None] == window_of(at_k[fk], shift)[None]
        want, tolerances = reference(q[fq].double(), k[fk].double(), v[fk].double(), do[fq].double(), same, heads, dh ** -0.5)
        for what, t, rows, w, tol in zip(('out', 'dq', 'dk', 'dv'), got, (fq, fq, fk, fk), want, tolerances(TWO_PARTS)):
            within(t[rows.cuda()], w, tol + e * w.abs(), f'{what} of frame {frame}')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('cross', [False, True])
@pytest.mark.parametrize('cells', [12, 20, 64])
def test_windows_listed_for_more_cells_than_there_are_rows(cells, cross, dtype):
    """Five rows in a window whose other cells hold numbers that are no rows, and the work list of that very grid: the list puts the
    window among those of `cells` tokens, and every row of it is written."""
    from tmae_amd import ops
    g = torch.Generator().manual_seed(cells)
    m, d = 5, 64

    def window():
        grid = torch.full((64,), -1, dtype=torch.int32)
        at = torch.randperm(64, generator=g)[:cells]
        grid[at] = torch.arange(cells, dtype=torch.int32) + m
        grid[at[:m]] = torch.arange(m, dtype=torch.int32)
        return grid.cuda()
    gq = window()
    gk = window() if cross else gq
    q, k, v, do = (torch.randn(m, d, generator=g).to(dtype) for _ in range(4))
    want, tolerances = reference(q.double(), k.double(), v.double(), do.double(), torch.ones(m, m, dtype=torch.bool), 4, 0.25)
    wl = ops.window_worklist(gq, gk, 1, 8, 8, False)
    for covered in (False, True):
        leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
        o = ops.win_attn_dot(*leaves, gq, gk, 4, 1, 8, 8, False, worklist=wl, covered=covered)
        grads = torch.autograd.grad(o, leaves, do.cuda())
        for what, got, w, t in zip(('out', 'dq', 'dk', 'dv'), (o, *grads), want, tolerances(half_step(dtype))):
            within(got, w, t, what)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('heads,dh', [(5, 16), (2, 32), (1, 64)])
def test_a_key_of_probability_zero_adds_nothing(heads, dh, dtype):
    """One key of every window has logits of -2^17 and less, so that its probabilities are 0, and V of the type's largest and lowest
    values: out is that of the other keys, and its own dV is 0."""
    from tmae_amd import ops
    g = torch.Generator().manual_seed(heads)
    ny, d = 40, heads * dh
    for count in (300, 900, 1600):
        grid, at = place([count], 1, ny, ny, g)
        win = window_of(at, False)
        masked = torch.zeros(count, dtype=torch.bool)
        for w in win.unique():
            rows = (win == w).nonzero()[:, 0]
            if rows.numel() > 1:
                masked[rows[torch.randint(rows.numel(), (1,), generator=g)]] = True
        q, k, v, do = (torch.randn(count, d, generator=g).to(dtype) for _ in range(4))
        q.view(count, heads, dh)[..., 3] = -2.0 ** 10
        k.view(count, heads, dh)[..., 3] = 0.0
        k.view(count, heads, dh)[masked, :, 3] = 2.0 ** 10
        v[masked] = torch.where(torch.rand(int(masked.sum()), d, generator=g) < 0.5, 1, -1).to(dtype) * torch.finfo(dtype).max
        gr = grid.cuda()
        same = (win[:, None] == win[None]) & ~masked[None]
        clean = v.double()
        clean[masked] = 0.0
        want, tolerances = reference(q.double(), k.double(), clean, do.double(), same, heads, dh ** -0.5)
        tols = tolerances(half_step(dtype))
        for worklist in (None, ops.window_worklist(gr, gr, 1, ny, ny, False)):
            leaf = v.cuda().requires_grad_()
            o = ops.win_attn_dot(q.cuda(), k.cuda(), leaf, gr, gr, heads, 1, ny, ny, False, worklist=worklist, covered=True)
            dv, = torch.autograd.grad(o, leaf, do.cuda())
            within(o, want[0], tols[0], 'out')
            within(dv, want[3], tols[3], 'dv')
            assert not dv[masked.cuda()].any()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('heads,dh', [(5, 16), (2, 32), (1, 64)])
def test_a_key_that_infinity_masks(heads, dh, dtype):
    """One key of every window holds an infinity where all queries are negative: its logits are -inf, its probabilities 0.  The results are
    those of the other keys: nothing of it reaches them over the slots behind a window's last query (0 times an infinity).  Its own dK and
    dV are 0, and only that channel of dQ (0 times the infinity) has no value."""
    from tmae_amd import ops
    g = torch.Generator().manual_seed(heads)
    ny, d = 40, heads * dh
    for count in (300, 900, 1600, 9 * 900):                                             # 1 to 64 tokens a window; one frame, or nine
        batch = max(1, count // 1600)
        count = count // batch
        grid, at = place([count] * batch, batch, ny, ny, g)
        win = window_of(at, False)
        n = at.shape[0]
        masked = torch.zeros(n, dtype=torch.bool)
        for w in win.unique():
            rows = (win == w).nonzero()[:, 0]
            if rows.numel() > 1:
                masked[rows[torch.randint(rows.numel(), (1,), generator=g)]] = True
        q, k, v, do = (torch.randn(n, d, generator=g).to(dtype) for _ in range(4))
        q[:, 3] = -q[:, 3].abs() - 0.125
        k[masked, 3] = float('inf')
        gr = grid.cuda()
        tail = at[:, 0] == batch - 1                                                    # a frame of them against the definition
        same = (win[tail][:, None] == win[tail][None]) & ~masked[tail][None]
        clean = k[tail].double()
        clean[masked[tail], 3] = 0.0
        # (of heads without the infinity the key is not masked: the first head alone)
        want, tolerances = reference(q[tail, :dh].double(), clean[:, :dh], v[tail, :dh].double(), do[tail, :dh].double(), same, 1, dh ** -0.5)
        for worklist in (None, ops.window_worklist(gr, gr, batch, ny, ny, False)):
            leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
            o = ops.win_attn_dot(*leaves, gr, gr, heads, batch, ny, ny, False, worklist=worklist, covered=True)
            grads = torch.autograd.grad(o, leaves, do.cuda())
            for what, got, w, t in zip(('out', 'dq', 'dk', 'dv'), (o, *grads), want, tolerances(half_step(dtype))):
                got = got.detach().cpu()
                channels = torch.arange(dh) if what != 'dq' else torch.tensor([c for c in range(dh) if c != 3])
                assert torch.isfinite(got[:, [c for c in range(d) if what != 'dq' or c != 3]]).all(), what
                within(got[tail][:, channels], w[:, channels], t[:, channels], what)


def test_frequencies_made_in_inference_mode_serve_training(monkeypatch):
    """The layer keeps its frequencies from the first call on; made in inference mode they would be refused by the first recorded one."""
    from types import SimpleNamespace
    from tmae_amd import ops
    from tmae_amd.modules.sst import WindowAttention
    seen = []
    monkeypatch.setattr(ops, 'rotary_axes', lambda heads, pos, f, sections: seen.append(f) or heads)
    a = WindowAttention(128, 8, 0.0, {'cosine': False, 'rotary': {'SECTIONS': [4, 4]}}).self_attn
    plan = SimpleNamespace(positions=lambda axes, time=0: torch.zeros(3, axes, dtype=torch.int32))
    with torch.inference_mode():
        a.turn(torch.zeros(3, 256), plan, True, True)
    a.turn(torch.zeros(3, 256, requires_grad=True), plan, True, True)
    assert len(seen) == 2 and not any(f.is_inference() for f in seen)
    assert torch.equal(seen[0], ops.rotary_freqs((4, 4), 100.0))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('heads,dh', [(5, 16), (2, 32), (1, 64)])
def test_an_infinite_gradient_of_a_probability_stays_one(heads, dh, dtype):
    """One query a window, V of one of its keys infinite in one channel: dP of that key is infinite, so is sum_j P dP, and dS of every other
    key is the opposite infinity: dK of those is that times the query, an infinity of a known sign in every channel of the head."""
    from tmae_amd import ops
    g = torch.Generator().manual_seed(heads)
    batch, ny, d = 2, 40, heads * dh
    for count in (300, 900, 1600):
        grid_k, at_k = place([count] * batch, batch, ny, ny, g)
        win = window_of(at_k, False)
        homes = win.unique()
        homes = homes[torch.tensor([int((win == w).sum()) > 1 for w in homes])]
        first = torch.stack([(win == w).nonzero()[0, 0] for w in homes])                # the query stands in the cell of a key
        grid_q = torch.full_like(grid_k, -1)
        grid_q[at_k[first, 0] * ny * ny + at_k[first, 1] * ny + at_k[first, 2]] = torch.arange(len(homes), dtype=torch.int32)
        mq, mk = len(homes), at_k.shape[0]
        q, do = (torch.randn(mq, d, generator=g).to(dtype) for _ in range(2))
        k, v = (torch.randn(mk, d, generator=g).to(dtype) for _ in range(2))
        bad = torch.stack([(win == w).nonzero()[-1, 0] for w in homes])
        v[bad, 3] = float('inf')
        of = torch.full((mk,), -1, dtype=torch.long)
        for i, w in enumerate(homes):
            of[win == w] = i
        rest = of >= 0
        rest[bad] = False
        sign = -torch.sign(do[of[rest], 3].float())[:, None] * torch.sign(q[of[rest], :dh].float())
        gq, gk = grid_q.cuda(), grid_k.cuda()
        for worklist in (None, ops.window_worklist(gq, gk, batch, ny, ny, False)):
            leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
            o = ops.win_attn_dot(*leaves, gq, gk, heads, batch, ny, ny, False, worklist=worklist, covered=True)
            dk, dv = (t.cpu().float() for t in torch.autograd.grad(o, leaves[1:], do.cuda()))
            assert torch.equal(dk[rest][:, :dh], sign * float('inf'))
            assert torch.isfinite(dk[:, dh:]).all() and torch.isfinite(dv).all()
