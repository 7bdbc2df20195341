"""Measured cases of the row operators: layer norm, counter-based dropout, and residual + dropout + layer norm.

Every operator works on rows: the last axis of x, `c` values wide, is normalised or masked; `pad` more values may lie between
two rows (a channel slice of wider pixel-major rows).  `run` is one pass as a training step or a serving call makes it: in
elementary torch operations where `own` is false, through `fiery_amd.row_ops` where it is true.

A dropped value is a function of (seed, call, row, column) alone.  Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random
numbers: as easy as 1, 2, 3", 2011) turns the counter (column // 8, row, call's low word, call's high word) under the key
(seed's low word, seed's high word) into four words; column c takes word (c % 8) // 2, its low half where c is even.  The value
is kept where that half is at least t = round(65536 p), and is then multiplied with 65536 / (65536 - t).  "channel" uses the
index along the first axis as the row, "sample" does too and takes column 0 for all.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def _norm(name, n, inner, c, dtype, train, pad=0, params=None):
    case = dict(op='layer_norm', n=n, inner=inner, c=c, pad=pad, dtype=dtype, params=params or dtype, train=train)
    return dict(case, name=name) if name else case


def _drop(name, n, inner, c, dtype, train, p, per='element', residual=False, stream=None, pad=0):
    case = dict(op='dropout', n=n, inner=inner, c=c, pad=pad, dtype=dtype, stream=stream or dtype, train=train, p=p, per=per, residual=residual)
    return dict(case, name=name) if name else case


def _join(name, n, inner, c, dtype, train, p, per='element', stream=None, params=None, pad=0):
    case = dict(op='dropout_add_layer_norm', n=n, inner=inner, c=c, pad=pad, dtype=dtype, stream=stream or dtype, params=params or dtype,
                train=train, p=p, per=per)
    return dict(case, name=name) if name else case


def listed():
    return [
        _norm('norm_token', 1, 1, 512, 'bf16', False),                    # serving, one row as wide as the lift head's features
        _norm('norm_images_f16', 54, 28 * 60, 128, 'f16', False),          # forward over 54 camera images at 1/8 resolution
        _norm('norm_bev_train', 12, 200 * 200, 64, 'f32', True),           # training step on 3 samples x 4 future BEV maps
        _norm('norm_odd_train', 6, 200 * 200, 35, 'bf16', True, params='f32'),   # the temporal blocks' 35-channel paths
        _norm('norm_wide_train', 8, 1024, 4096, 'bf16', True),             # wide rows: sequences of 1024 with 4096 features
        _drop('drop_token', 1, 1, 512, 'f32', False, 0.1),                 # smallest call
        _drop('drop_channel_train', 12, 200 * 200, 64, 'f32', True, 0.1, per='channel', residual=True),   # a Bottleneck's Dropout2d + skip
        _drop('drop_wide_train', 16, 1024, 4096, 'bf16', True, 0.25),      # element masks, where the generator costs the most
        _drop('drop_sample_train', 54, 28 * 60, 56, 'f32', True, 0.125, per='sample', residual=True),     # the trunk's drop-connect + skip
        _join('join_small_train', 3, 11, 200, 'f16', True, 0.1),           # few rows of an odd count
        _join('join_bev_train', 12, 200 * 200, 64, 'f32', True, 0.2, per='sample'),      # stochastic depth on the BEV maps
        _join('join_wide_train', 8, 1024, 4096, 'bf16', True, 0.1),        # residual, dropout and norm between wide layers
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(('layer_norm', 'dropout', 'dropout_add_layer_norm'))
    c = spread(1 if op == 'dropout' else 4, 8192)
    rows = spread(1, min(480000, 30_000_000 // c))
    n = spread(1, rows)
    inner, dtype, train = max(1, rows // n), rng.choice(('f32', 'bf16', 'f16')), rng.random() < 0.7
    pad, p, per = rng.choice((0, 0, 1, 5, 8)), round(rng.uniform(0.02, 0.9), 3), rng.choice(('element', 'element', 'channel', 'sample'))
    wide = rng.random() < 0.5                                              # 32-bit stream and parameters beside 16-bit rows
    if op == 'layer_norm':
        return _norm(None, n, inner, c, dtype, train, pad, 'f32' if wide else None)
    if op == 'dropout':
        skip = rng.random() < 0.5 or per != 'element' or n * inner * c < 64    # whole samples and channels are dropped beside a skip
        return _drop(None, n, inner, c, dtype, train, p, per, skip, None, pad)
    return _join(None, n, inner, c, dtype, train, p, per, 'f32' if wide else None, 'f32' if wide else None, pad)


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    shape, dtype, train = (case['n'], case['inner'], case['c']), TYPES[case['dtype']], case['train']

    def rows(kind, pad=0, spread=1.0):
        wide = torch.empty(shape[0], shape[1], shape[2] + pad, dtype=kind, device='cuda').normal_(0.3, spread, generator=gen)
        return wide[..., :shape[2]]

    s = dict(case=case, x=rows(dtype, case['pad'], 1.5).detach().requires_grad_(train))
    if 'params' in case:
        kind = TYPES[case['params']]
        s['weight'] = torch.empty(shape[2], dtype=kind, device='cuda').normal_(1.0, 0.2, generator=gen).requires_grad_(train)
        s['bias'] = torch.empty(shape[2], dtype=kind, device='cuda').normal_(0.0, 0.2, generator=gen).requires_grad_(train)
    if case['op'] == 'dropout_add_layer_norm' or case.get('residual'):
        s['residual'] = rows(TYPES[case['stream']]).detach().requires_grad_(train)
    if 'p' in case:
        s['rng'] = torch.empty(2, dtype=torch.int64, device='cuda').random_(generator=gen)     # [seed, call], on the device
    if train:
        s['dy'] = rows(TYPES[case['stream']] if case['op'] == 'dropout' else dtype)
        if case['op'] == 'dropout_add_layer_norm':
            s['dh'] = rows(TYPES[case['stream']])
    return s


# ---- the plain form: elementary torch operations in 32 bits -------------------------------------------------------------
def _keep(case, rng):
    """Truth values of what is kept, shaped to broadcast against x."""
    n, inner, c, low = case['n'], case['inner'], case['c'], 0xffffffff
    rows = n * inner if case['per'] == 'element' else n
    width = 1 if case['per'] == 'sample' else c
    groups = (width + 7) // 8
    a = torch.arange(groups, device=rng.device).expand(rows, groups)
    b = torch.arange(rows, device=rng.device).unsqueeze(1).expand(rows, groups)
    d, e = rng[1] & low, (rng[1] >> 32) & low
    k0, k1 = rng[0] & low, (rng[0] >> 32) & low
    for _ in range(10):
        p, q = a * 0xD2511F53, d * 0xCD9E8D57                              # products modulo 2^64: all their bits are there
        a, b, d, e = (q >> 32 & low) ^ b ^ k0, q & low, (p >> 32 & low) ^ e ^ k1, p & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    words = torch.stack(torch.broadcast_tensors(a, b, d, e), -1)
    halves = torch.stack((words & 0xffff, words >> 16), -1).view(rows, groups * 8)[:, :width]
    keep = halves >= round(65536 * case['p'])
    return keep.view(n, inner, c) if case['per'] == 'element' else keep.view(n, 1, width)


def _scale(case):
    t = round(65536 * case['p'])
    return 65536.0 / (65536 - t) if t < 65536 else 0.0


def _plain(s):
    case, x = s['case'], s['x'].float()
    out, keep, h = {}, None, x
    if 'p' in case:
        keep = _keep(case, s['rng'])
        h = torch.where(keep, x * _scale(case), 0.0)
        if 'residual' in s:
            h = s['residual'].float() + h
    if case['op'] == 'dropout':
        out['y'] = h.to(TYPES[case['stream']])
        if case['train']:
            dh = s['dy'].float()
    else:
        w = s['weight'].float()
        centred = h - h.mean(-1, keepdim=True)
        rstd = 1.0 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
        xhat = centred * rstd
        out['y'] = (xhat * w + s['bias'].float()).to(s['x'].dtype)
        if keep is not None:
            out['h'] = h.to(TYPES[case['stream']])
        if case['train']:
            g = s['dy'].float()
            gw = g * w
            dh = rstd * (gw - gw.mean(-1, keepdim=True) - xhat * (gw * xhat).mean(-1, keepdim=True))
            if keep is not None:
                dh = dh + s['dh'].float()
            out['dweight'] = (g * xhat).sum((0, 1)).to(s['weight'].dtype)
            out['dbias'] = g.sum((0, 1)).to(s['bias'].dtype)
    if case['train']:
        out['dx'] = (dh if keep is None else torch.where(keep, dh * _scale(case), 0.0)).to(s['x'].dtype)
        if 'residual' in s:
            out['dresidual'] = dh.to(s['residual'].dtype)
    return out


# ---- the framework's calls ---------------------------------------------------------------------------------------------
def _calls(s):
    from fiery_amd import row_ops
    case, x = s['case'], s['x']
    if case['op'] == 'layer_norm':
        y = row_ops.layer_norm(x, s['weight'], s['bias'], EPS)
        if not case['train']:
            return {'y': y}
        dx, dw, db = torch.autograd.grad(y, (x, s['weight'], s['bias']), s['dy'])
        return {'y': y, 'dx': dx, 'dweight': dw, 'dbias': db}
    if case['op'] == 'dropout':
        residual = s.get('residual')
        y = row_ops.dropout(x, case['p'], s['rng'], per=case['per'], residual=residual)
        if not case['train']:
            return {'y': y}
        if residual is None:
            return {'y': y, 'dx': torch.autograd.grad(y, x, s['dy'])[0]}
        dx, dr = torch.autograd.grad(y, (x, residual), s['dy'])
        return {'y': y, 'dx': dx, 'dresidual': dr}
    # (gradients at h before its rounding, as the definition has them)
    y, h = row_ops.dropout_add_layer_norm(x, s['residual'], s['weight'], s['bias'], case['p'], s['rng'], per=case['per'], eps=EPS, keep='inputs')
    if not case['train']:
        return {'y': y, 'h': h}
    dx, dr, dw, db = torch.autograd.grad((y, h), (x, s['residual'], s['weight'], s['bias']), (s['dy'], s['dh']))
    return {'y': y, 'h': h, 'dx': dx, 'dresidual': dr, 'dweight': dw, 'dbias': db}


def run(state):
    if own:
        return _calls(state)
    with torch.no_grad():
        return _plain(state)


def work(case):
    """Bytes: each input read once, each output written once.  Flops: the floating-point operations of the formulas."""
    rows, c = case['n'] * case['inner'], case['c']
    size = {'f32': 4, 'bf16': 2, 'f16': 2}
    x, n = size[case['dtype']], rows * c
    if case['op'] == 'layer_norm':
        w = size[case['params']] * c
        return {'bytes': (5 if case['train'] else 2) * n * x + (5 if case['train'] else 2) * w, 'flops': (22 if case['train'] else 8) * n}
    stream = size[case['stream']]
    if case['op'] == 'dropout':
        forward = x + (2 * stream if case['residual'] else x)
        backward = (stream + x + (stream if case['residual'] else 0)) if case['train'] else 0
        return {'bytes': n * (forward + backward) + 16, 'flops': (3 if case['train'] else 2) * n}
    w = size[case['params']] * c
    forward, backward = 2 * x + 2 * stream, 2 * x + 2 * stream                 # x, residual -> y, h; dy, dh -> dx, dresidual (h is at hand)
    return {'bytes': n * (forward + (backward + stream if case['train'] else 0)) + 5 * w + 16, 'flops': (26 if case['train'] else 10) * n}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------
def _halves(row, columns, seed, call):
    """The 16-bit numbers of `columns` consecutive columns of the rows `row` (an array), as the definition reads them."""
    mask, shift = np.uint64(0xffffffff), np.uint64(32)
    count = (columns + 7) // 8
    ctr = [np.broadcast_to(np.arange(count, dtype=np.uint64), (row.size, count)), np.broadcast_to(row.astype(np.uint64)[:, None], (row.size, count)),
           np.full((row.size, count), call & 0xffffffff, np.uint64), np.full((row.size, count), call >> 32, np.uint64)]
    for i in range(10):
        key = [np.uint64(((seed & 0xffffffff) + i * 0x9E3779B9) % 2 ** 32), np.uint64(((seed >> 32) + i * 0xBB67AE85) % 2 ** 32)]
        left, right = np.uint64(0xD2511F53) * ctr[0], np.uint64(0xCD9E8D57) * ctr[2]
        ctr = [(right >> shift) ^ ctr[1] ^ key[0], right & mask, (left >> shift) ^ ctr[3] ^ key[1], left & mask]
    words = np.stack([w.astype(np.uint32) for w in ctr], -1)
    return np.stack([words & 0xffff, words >> 16], -1).reshape(row.size, count * 8)[:, :columns].astype(np.int32)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        f = {k: v.detach().double() for k, v in s.items() if k not in ('case', 'rng')}
        c, out, factor = case['c'], {}, None
        h = f['x']
        if 'p' in case:
            number, call = (int(v) % 2 ** 64 for v in s['rng'].tolist())
            total, width = (case['n'] * case['inner'], c) if case['per'] == 'element' else (case['n'], 1 if case['per'] == 'sample' else c)
            step = max(1, 2 ** 16 // ((width + 7) // 8))                       # rows at a time: the words stay in the processor's cache
            drawn = np.concatenate([_halves(np.arange(i, min(i + step, total)), width, number, call) for i in range(0, total, step)])
            border = int(np.rint(case['p'] * 2 ** 16))
            factor = torch.from_numpy(drawn >= border).to(h.device).double() * (2 ** 16 / max(1, 2 ** 16 - border))
            factor = factor.view(case['n'], -1, width)
            h = h * factor + f.get('residual', 0.0)
        if case['op'] == 'dropout':
            back = f.get('dy')
            out['y'] = h
        else:
            mean = h.sum(-1, keepdim=True) / c
            deviation = torch.sqrt(((h - mean) ** 2).sum(-1, keepdim=True) / c + EPS)
            unit = (h - mean) / deviation
            out['y'] = unit * f['weight'] + f['bias']
            if factor is not None:
                out['h'] = h
            if case['train']:
                inner = f['dy'] * f['weight']
                back = (inner * c - inner.sum(-1, keepdim=True) - unit * (inner * unit).sum(-1, keepdim=True)) / (c * deviation)
                back = back + f.get('dh', 0.0)
                out['dweight'], out['dbias'] = (f['dy'] * unit).sum((0, 1)), f['dy'].sum((0, 1))
        if case['train']:
            out['dx'] = back if factor is None else back * factor
            if 'residual' in f:
                out['dresidual'] = back
    return out
