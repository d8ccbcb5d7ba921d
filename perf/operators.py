"""The attention operators of the encoder layers as cases: rotary positions with several axes, the norms of queries and keys with
the rotation in the same pass, and scaled-dot-product attention inside 8x8 windows.

The shapes are those of this framework's encoder: tokens are the occupied cells of a bird's-eye grid (468 x 468 at stage 1,
234 x 234 at stage 2, eight frames a step, about 47 k cells a frame), 8 heads of 16 (d 128) or 32 (d 256) channels, positions
(time, y, x).  `own` false: elementary torch operations in float32; true: the calls a user makes of tmae_amd.ops."""
import math
import os
import sys

import numpy as np
import torch

own = False

EPS = 1e-6
BASE = 100.0


def _ops():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 't-mae_amd')
    if root not in sys.path:
        sys.path.insert(0, root)
    from tmae_amd import ops
    return ops


def _dtype(case):
    return {'bf16': torch.bfloat16, 'f32': torch.float32}[case['dtype']]


def _sections(case):
    return tuple(int(s) for s in case['sections'].split('+'))


# ------------------------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one token's queries and keys (8 + 8 heads of 32) on their way into an attention: latency
        dict(name='rotary_one_token', op='rotary', n=1, heads=16, spare=0, dh=32, sections='4+6+6', interleaved=False, far=False,
             dtype='bf16', train=False),
        # stage 1, eight frames: the packed q | k out of a packed q | k | v projection, forward and backward
        dict(name='rotary_stage1_train', op='rotary', n=375413, heads=16, spare=8, dh=16, sections='4+4', interleaved=False,
             far=False, dtype='bf16', train=True),
        # one float32 frame, odd head count and width, pass-through channels, adjacent pairs, far positions (time stamps)
        dict(name='rotary_far_f32', op='rotary', n=51237, heads=7, spare=0, dh=40, sections='4+6+6', interleaved=True, far=True,
             dtype='f32', train=False),
        # a handful of tokens at inference: latency
        dict(name='qk_norm_few', op='qk_norm', n=7, hq=8, hk=8, dh=32, sections='4+6+6', interleaved=False, per_head=False,
             dtype='bf16', train=False),
        # stage 1 training, eight frames
        dict(name='qk_norm_stage1_train', op='qk_norm', n=375413, hq=8, hk=8, dh=16, sections='4+4', interleaved=False,
             per_head=False, dtype='bf16', train=True),
        # stage 2 training, three axes
        dict(name='qk_norm_stage2_train', op='qk_norm', n=131072, hq=8, hk=8, dh=32, sections='4+6+6', interleaved=False,
             per_head=False, dtype='bf16', train=True),
        # float32, fewer key heads than query heads, a gain for each head, a width that is no power of two
        dict(name='qk_norm_shared_keys_f32', op='qk_norm', n=20011, hq=12, hk=4, dh=72, sections='12+12+12', interleaved=True,
             per_head=True, dtype='f32', train=True),
        # a small scene at inference: latency
        dict(name='attn_small_scene', op='attn', batch=1, ny=24, nx=24, nq=97, nk=0, heads=8, dh=16, shift=False, dtype='bf16',
             train=False),
        # stage 1 self-attention, eight frames, forward and backward: the largest
        dict(name='attn_stage1_train', op='attn', batch=8, ny=468, nx=468, nq=46927, nk=0, heads=8, dh=16, shift=False,
             dtype='bf16', train=True),
        # stage 2 cross-attention: a quarter of the current frame's cells against the previous frame's, shifted windows
        dict(name='attn_stage2_cross_train', op='attn', batch=8, ny=234, nx=234, nq=4097, nk=16381, heads=8, dh=32, shift=True,
             dtype='bf16', train=True),
        # one float32 frame of stage 2, forward and backward
        dict(name='attn_frame_f32_train', op='attn', batch=1, ny=234, nx=234, nq=16381, nk=0, heads=8, dh=32, shift=True,
             dtype='f32', train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['rotary', 'qk_norm', 'attn'])
    dtype = rng.choice(['bf16', 'bf16', 'f32'])
    train = rng.random() < 0.6
    if op in ('rotary', 'qk_norm'):
        dh = rng.choice([16, 24, 32, 40, 64, 72, 96, 128])
        axes = rng.choice([1, 2, 3])
        most = dh // 2 // axes
        sections = '+'.join(str(rng.randint(1, most)) for _ in range(axes))
        hq, hk = rng.randint(1, 12), rng.randint(1, 12)
        widest = 90_000_000 if dtype == 'bf16' else 45_000_000          # elements: the largest listed one has 96 M, in bf16
        n = _log_int(rng, 1, max(1, min(375413, widest // ((hq + hk + 8) * dh))))
        case = dict(op=op, n=n, dh=dh, sections=sections, interleaved=rng.random() < 0.5, dtype=dtype, train=train)
        if op == 'rotary':
            case.update(heads=hq + hk, spare=rng.choice([0, 1, 8]), far=rng.random() < 0.3)
        else:
            case.update(hq=hq, hk=hk, per_head=rng.random() < 0.3)
        return case
    dh = rng.choice([16, 32, 64])
    heads = rng.randint(1, 8 if dh < 64 else 4)
    ny, nx = _log_int(rng, 1, 468), _log_int(rng, 1, 468)
    widest = 220_000_000 if dtype == 'bf16' else 110_000_000            # cells x channels: the largest listed one has 224 M, in bf16
    batch = rng.randint(1, max(1, min(8, widest // (heads * dh * ny * nx))))
    share = rng.choice([0.02, 0.08, 0.2, 0.5, 1.0]) if ny * nx * batch * heads * dh < widest // 8 else rng.choice([0.02, 0.08, 0.2])
    nq = max(1, int(ny * nx * share * rng.uniform(0.7, 1.0)))
    case = dict(op=op, batch=batch, ny=ny, nx=nx, nq=nq, nk=0, heads=heads, dh=dh, shift=rng.random() < 0.5, dtype=dtype, train=train)
    if rng.random() < 0.4:
        case.update(nk=max(1, int(ny * nx * rng.uniform(0.02, share))))
    return case


# ----------------------------------------------------------------------------------------------------------------- inputs

def _density(ny, nx):
    """How likely a cell of a square scene is to hold points: 1 / r^2 around the sensor, flat within 2 m (edge 149.76 m)."""
    y = (np.arange(ny) + 0.5 - ny / 2) * (149.76 / max(ny, nx))
    x = (np.arange(nx) + 0.5 - nx / 2) * (149.76 / max(ny, nx))
    return 1.0 / np.maximum(y[:, None] ** 2 + x[None, :] ** 2, 4.0)


def _tokens(case, n_frame, g):
    """n_frame occupied cells of every frame, drawn by that density without replacement (the order of exponential clocks), as sorted
    rows: indices [n, 3] (frame, y, x) and the dense grid of row numbers, -1 where a cell is empty."""
    b, ny, nx = case['batch'], case['ny'], case['nx']
    w = torch.from_numpy(_density(ny, nx).reshape(-1)).cuda()
    clocks = -torch.log(torch.rand((b, ny * nx), generator=g, device='cuda', dtype=torch.float64)) / w
    cells = clocks.topk(n_frame, dim=1, largest=False).indices.sort(dim=1).values
    flat = (cells + torch.arange(b, device='cuda')[:, None] * (ny * nx)).reshape(-1)
    grid = torch.full((b * ny * nx,), -1, dtype=torch.int32, device='cuda')
    grid[flat] = torch.arange(flat.numel(), dtype=torch.int32, device='cuda')
    cells = cells.reshape(-1)
    frame = torch.arange(b, device='cuda').repeat_interleave(n_frame)
    return torch.stack([frame, cells // nx, cells % nx], 1).int().contiguous(), grid


def _windows(grid, case):
    """[windows, 64] row numbers, -1 where a cell is empty: windows start a whole (or, shifted, half) a window before the grid."""
    b, ny, nx = case['batch'], case['ny'], case['nx']
    wy, wx = -(-ny // 8) + 1, -(-nx // 8) + 1
    s = 4 if case['shift'] else 8
    canvas = torch.full((b, wy * 8, wx * 8), -1, dtype=torch.int64, device=grid.device)
    canvas[:, s:s + ny, s:s + nx] = grid.view(b, ny, nx)
    return canvas.view(b, wy, 8, wx, 8).permute(0, 1, 3, 2, 4).reshape(-1, 64)


def _slots(rows, n):
    """For each token its place in the flattened window table."""
    at = torch.empty((n,), dtype=torch.int64, device=rows.device)
    there = (rows.reshape(-1) >= 0).nonzero().squeeze(1)
    at[rows.reshape(-1)[there]] = there
    return at


def _inv_freq(case):
    """Each axis has its own ladder of frequencies, base^(-j/p), as float64."""
    return torch.cat([BASE ** (-torch.arange(p, dtype=torch.float64) / p) for p in _sections(case)]).cuda()


def _positions(n, case, g):
    axes = len(_sections(case))
    if case.get('far'):          # time stamps and far cells: whole numbers up to 2^23, on either side
        return torch.randint(-(1 << 23), 1 << 23, (n, axes), generator=g, device='cuda', dtype=torch.int32)
    return torch.randint(0, 468, (n, axes), generator=g, device='cuda', dtype=torch.int32)


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dt = _dtype(case)

    def rand(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device='cuda') * scale).to(dt)

    def gain(heads):
        shape = (heads, case['dh']) if case.get('per_head') else (case['dh'],)
        return 1.0 + 0.2 * torch.randn(shape, generator=g, device='cuda')

    s = dict(case=case)
    if case['op'] in ('rotary', 'qk_norm'):
        n, dh = case['n'], case['dh']
        s['inv_freq'] = _inv_freq(case)
        s['positions'] = _positions(n, case, g)
        if case['op'] == 'rotary':
            # `spare`: the heads behind the rotated ones in the rows of a packed projection
            s['x'] = rand(n, case['heads'] + case['spare'], dh)[:, :case['heads']]
            s['dy'] = rand(n, case['heads'], dh) if case['train'] else None
        else:
            s['x'] = rand(n, case['hq'] + case['hk'], dh, scale=1.5)
            s['dy'] = rand(n, case['hq'] + case['hk'], dh) if case['train'] else None
            s['q_gain'], s['k_gain'] = gain(case['hq']), gain(case['hk'])
        return s
    d = case['heads'] * case['dh']
    indices, grid = _tokens(case, case['nq'], g)
    n = indices.shape[0]
    s['grid_q'] = grid
    rows_q = _windows(grid, case)
    if case['nk']:
        _, s['grid_k'] = _tokens(case, case['nk'], g)
        nk = case['batch'] * case['nk']
        rows_k = _windows(s['grid_k'], case)
        used = ((rows_q >= 0) | (rows_k >= 0)).any(1)
        s['rows_q'], s['rows_k'] = rows_q[used], rows_k[used]
        s['slots_q'], s['slots_k'] = _slots(s['rows_q'], n), _slots(s['rows_k'], nk)
        s['q'], s['k'], s['v'] = rand(n, d), rand(nk, d), rand(nk, d)
    else:
        s['grid_k'] = grid
        s['rows_q'] = s['rows_k'] = rows_q[(rows_q >= 0).any(1)]
        s['slots_q'] = s['slots_k'] = _slots(s['rows_q'], n)
        s['qk'], s['v'] = rand(n, 2 * d), rand(n, d)
    s['do'] = rand(n, d) if case['train'] else None
    if own:      # the list of occupied windows that a program builds once for a set of tokens, as the table above for the plain form
        s['worklist'] = _ops().window_worklist(s['grid_q'], s['grid_k'], case['batch'], case['ny'], case['nx'], case['shift'])
    return s


# ------------------------------------------------------------------------------------------------------------ plain forms

def _cos_sin(s):
    sections = _sections(s['case'])
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(s['positions'].device)
    theta = s['positions'].double()[:, axis] * s['inv_freq']
    return theta.cos().float()[:, None], theta.sin().float()[:, None]


def _turn(x, cos, sin, interleaved):
    """x [n, h, dh] float32, the first 2P channels turned by the angles."""
    p = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * p:2], x[..., 1:2 * p:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :p], x[..., p:2 * p]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, x[..., 2 * p:]], -1)


def _plain_rotary(s):
    c = s['case']
    cos, sin = _cos_sin(s)
    y = _turn(s['x'].float(), cos, sin, c['interleaved']).to(s['x'].dtype)
    if not c['train']:
        return [y]
    return [y, _turn(s['dy'].float(), cos, -sin, c['interleaved']).to(s['x'].dtype)]


def _gains(s, hq, hk):
    dh = s['case']['dh']
    return torch.cat([s['q_gain'].expand(hq, dh), s['k_gain'].expand(hk, dh)])


def _norm_turn(x, gains, cos, sin, interleaved):
    x = x.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return _turn(x * r * gains, cos, sin, interleaved)


def _norm_turn_backward(x, dy, gains, cos, sin, interleaved):
    x = x.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    xh = x * r
    dz = _turn(dy.float(), cos, -sin, interleaved)
    t = dz * gains
    dx = r * (t - xh * (t * xh).mean(-1, keepdim=True))
    return dx, (dz * xh).sum(0, dtype=torch.float64)                    # the sum is long: over every token


def _split_gain_gradient(dgain, hq, like):
    dq, dk = dgain[:hq], dgain[hq:]
    if like.dim() == 1:
        dq, dk = dq.sum(0), dk.sum(0)
    return dq.float(), dk.float()


def _plain_qk_norm(s):
    c = s['case']
    cos, sin = _cos_sin(s)
    gains = _gains(s, c['hq'], c['hk'])
    y = _norm_turn(s['x'], gains, cos, sin, c['interleaved']).to(s['x'].dtype)
    if not c['train']:
        return [y]
    dx, dgain = _norm_turn_backward(s['x'], s['dy'], gains, cos, sin, c['interleaved'])
    return [y, dx.to(s['x'].dtype), *_split_gain_gradient(dgain, c['hq'], s['q_gain'])]


def _plain_attention(s, q, k, v, do):
    """q, k, v, do: [tokens, d] -> the rows of the output and, where do is given, of the gradients, in the inputs' type."""
    c = s['case']
    h, dh = c['heads'], c['dh']
    scale = dh ** -0.5
    dt = q.dtype

    def into(t, rows):        # [tokens, d] -> [windows, heads, 64, dh], zeros where there is no token
        t = t.float()[rows.clamp(min=0)] * (rows >= 0)[..., None]
        return t.view(-1, 64, h, dh).transpose(1, 2).contiguous()

    def back(t, slots):
        return t.transpose(1, 2).reshape(-1, h * dh)[slots].to(dt)

    there = (s['rows_k'] >= 0)[:, None, None, :]
    qw, kw, vw = into(q, s['rows_q']), into(k, s['rows_k']), into(v, s['rows_k'])
    logits = torch.matmul(qw, kw.transpose(2, 3)) * scale
    logits = torch.where(there, logits, torch.full_like(logits, -math.inf))
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    out = back(torch.matmul(p, vw), s['slots_q'])
    if do is None:
        return [out]
    dow = into(do, s['rows_q'])
    dv = torch.matmul(p.transpose(2, 3), dow)
    dp = torch.matmul(dow, vw.transpose(2, 3))
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(ds, kw)
    dk = torch.matmul(ds.transpose(2, 3), qw)
    return [out, back(dq, s['slots_q']), back(dk, s['slots_k']), back(dv, s['slots_k'])]


def _plain_attn(s):
    if s['case']['nk']:
        return _plain_attention(s, s['q'], s['k'], s['v'], s['do'])
    d = s['v'].shape[1]
    got = _plain_attention(s, s['qk'][:, :d], s['qk'][:, d:], s['v'], s['do'])
    return got if len(got) == 1 else [got[0], torch.cat([got[1], got[2]], 1), got[3]]


# -------------------------------------------------------------------------------------------------------- the framework's

def _leaf(t, train):
    return t.detach().requires_grad_() if train else t


def _own(s):
    ops = _ops()
    c = s['case']
    train = c['train']
    if c['op'] == 'rotary':
        x = _leaf(s['x'], train)
        y = ops.rotary_axes(x, s['positions'], s['inv_freq'], _sections(c), interleaved=c['interleaved'])
        return [y.detach(), *torch.autograd.grad(y, x, s['dy'])] if train else [y]
    if c['op'] == 'qk_norm':
        x, gq, gk = (_leaf(s[k], train) for k in ('x', 'q_gain', 'k_gain'))
        y = ops.qk_norm_rotary(x, gq, gk, s['positions'], s['inv_freq'], _sections(c), q_heads=c['hq'], eps=EPS,
                               interleaved=c['interleaved'])
        return [y.detach(), *torch.autograd.grad(y, (x, gq, gk), s['dy'])] if train else [y]
    grids = (s['grid_q'], s['grid_k'], c['heads'], c['batch'], c['ny'], c['nx'], c['shift'])
    if c['nk']:
        q, k, v = (_leaf(s[n], train) for n in 'qkv')
        o = ops.win_attn_dot(q, k, v, *grids, worklist=s['worklist'], covered=True)
        return [o.detach(), *torch.autograd.grad(o, (q, k, v), s['do'])] if train else [o]
    qk, v = _leaf(s['qk'], train), _leaf(s['v'], train)
    o = ops.win_attn_dot(qk, v, None, *grids, worklist=s['worklist'], covered=True)
    return [o.detach(), *torch.autograd.grad(o, (qk, v), s['do'])] if train else [o]


def run(s):
    if own:
        return _own(s)
    return {'rotary': _plain_rotary, 'qk_norm': _plain_qk_norm, 'attn': _plain_attn}[s['case']['op']](s)


# ------------------------------------------------------------------------------------------------------------------- work

def _pairs(case):
    """Expected number of (query, key) pairs that share a window: a cell is drawn with probability 1 - exp(-t density)."""
    ny, nx = case['ny'], case['nx']
    dens = _density(ny, nx)

    def chance(n):
        lo, hi = 0.0, 1.0
        while (1 - np.exp(-hi * dens)).sum() < n - 1e-6 and hi < 1e12:
            hi *= 2
        for _ in range(60):
            mid = (lo + hi) / 2
            lo, hi = (mid, hi) if (1 - np.exp(-mid * dens)).sum() < n else (lo, mid)
        return 1 - np.exp(-hi * dens)

    s = 4 if case['shift'] else 8
    wy, wx = -(-ny // 8) + 1, -(-nx // 8) + 1

    def by_window(t):
        full = np.zeros((wy * 8, wx * 8))
        full[s:s + ny, s:s + nx] = t
        return full.reshape(wy, 8, wx, 8).sum((1, 3))

    p = chance(case['nq'])
    if case['nk']:
        return case['batch'] * float((by_window(p) * by_window(chance(case['nk']))).sum())
    return case['batch'] * float((by_window(p) ** 2 + by_window(p * (1 - p))).sum())


def work(case):
    es = 2 if case['dtype'] == 'bf16' else 4
    train = case['train']
    if case['op'] in ('rotary', 'qk_norm'):
        n, norm = case['n'], case['op'] == 'qk_norm'
        heads = case['hq'] + case['hk'] if norm else case['heads']
        rows, p = float(n) * heads * case['dh'], sum(_sections(case))
        turn = 6.0 * n * heads * p
        # in and out; for training the gradient in and out as well (a norm's input read once for both directions)
        b = 2 * rows * es * (2 if train else 1) + 4 * n * len(_sections(case)) + 8 * p
        f = turn * (2 if train else 1) + ((5 + (9 if train else 0)) * rows if norm else 0)
        return dict(bytes=b, flops=f)
    d = case['heads'] * case['dh']
    mq, mk = case['batch'] * case['nq'], case['batch'] * (case['nk'] or case['nq'])
    pairs = _pairs(case) * d
    b = es * d * (2.0 * mq + 2.0 * mk) + 4 * case['batch'] * case['ny'] * case['nx'] * (2 if case['nk'] else 1)
    if train:
        b += es * d * (2.0 * mq + 2.0 * mk)          # do in; dq, dk, dv out
    return dict(bytes=b, flops=pairs * (14 if train else 4))


# ------------------------------------------------------------------------------------------------------------------ exact

def _exact_turn(x, s, sign=1):
    """Complex multiplication in complex128."""
    c = s['case']
    sections = _sections(c)
    p = sum(sections)
    parts = torch.split(s['inv_freq'], sections)
    theta = torch.cat([s['positions'][:, a:a + 1].double() * w for a, w in enumerate(parts)], 1)
    e = torch.polar(torch.ones_like(theta), sign * theta)[:, None]
    head, rest = x[..., :2 * p], x[..., 2 * p:]
    z = torch.view_as_complex(head.reshape(*head.shape[:-1], p, 2).contiguous()) if c['interleaved'] \
        else torch.complex(head[..., :p], head[..., p:])
    z = torch.view_as_real(z * e)
    z = z.flatten(-2) if c['interleaved'] else torch.cat([z[..., 0], z[..., 1]], -1)
    return torch.cat([z, rest], -1)


def _exact_norm(x, gq, gk, hq):
    unit = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS)
    return torch.cat([unit[:, :hq] * gq, unit[:, hq:] * gk], 1)


def _exact_attention(q, k, v, s):
    """Frame after frame on the dense scene: every window of the scene's cells, empty ones included, with a bias of -inf."""
    c = s['case']
    h, dh, ny, nx = c['heads'], c['dh'], c['ny'], c['nx']
    at = 4 if c['shift'] else 8
    wy, wx = -(-ny // 8) + 1, -(-nx // 8) + 1
    gq, gk = s['grid_q'].view(-1, ny, nx), s['grid_k'].view(-1, ny, nx)

    def scene(t, g):
        dense = torch.zeros((wy * 8, wx * 8, h, dh), dtype=torch.float64, device=g.device)
        y, x = (g >= 0).nonzero(as_tuple=True)
        dense = dense.index_put((y + at, x + at), t[g[y, x].long()].view(-1, h, dh))
        return dense.view(wy, 8, wx, 8, h, dh).permute(0, 2, 4, 1, 3, 5).reshape(wy * wx, h, 64, dh)

    out = torch.zeros_like(q)
    for b in range(c['batch']):
        held = torch.zeros((wy * 8, wx * 8), dtype=torch.bool, device=q.device)
        held[at:at + ny, at:at + nx] = gk[b] >= 0
        held = held.view(wy, 8, wx, 8).permute(0, 2, 1, 3).reshape(wy * wx, 64)
        some = held.any(1)
        bias = torch.zeros(held.shape, dtype=torch.float64, device=q.device).masked_fill(~held & some[:, None], -math.inf)
        w = torch.softmax(scene(q, gq[b]) @ scene(k, gk[b]).transpose(-1, -2) / math.sqrt(dh) + bias[:, None, None], -1)
        o = (w * some[:, None, None, None]) @ scene(v, gk[b])
        o = o.view(wy, wx, h, 8, 8, dh).permute(0, 3, 1, 4, 2, 5).reshape(wy * 8, wx * 8, h * dh)
        y, x = (gq[b] >= 0).nonzero(as_tuple=True)
        out = out.index_put((gq[b][y, x].long(),), o[y + at, x + at])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    c = s['case']
    if c['op'] == 'rotary':
        y = _exact_turn(s['x'].double(), s)
        return [y, _exact_turn(s['dy'].double(), s, -1)] if c['train'] else [y]
    names = ['x', 'q_gain', 'k_gain'] if c['op'] == 'qk_norm' else ['q', 'k', 'v'] if c['nk'] else ['qk', 'v']
    leaves = {n: s[n].double().requires_grad_(c['train']) for n in names}
    if c['op'] == 'qk_norm':
        out = _exact_turn(_exact_norm(leaves['x'], leaves['q_gain'], leaves['k_gain'], c['hq']), s)
        dy = s['dy']
    else:
        d = c['heads'] * c['dh']
        dy = s['do']
        if c['nk']:
            q, k = leaves['q'], leaves['k']
        else:
            q, k = leaves['qk'][:, :d], leaves['qk'][:, d:]
        out = _exact_attention(q, k, leaves['v'], s)
    if not c['train']:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, [leaves[n] for n in names], dy.double())]
