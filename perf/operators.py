"""What group normalisation with an activation and activation checkpoints in 8 bits are measured on: the convolution blocks and
dense layers of the Darcy model in training, from one sample of the coarsest grid to full batches.

A case is a dict of plain values.  `run` computes an operator in its plain form, elementary torch operations in 32 bits, or, where
`own` is set, calls the framework.
"""
import math

import torch

own = False

TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
BYTES = {'fp32': 4, 'bf16': 2, 'fp16': 2}
BLOCK = 32                        # values that share a step in a checkpoint


def _norm(kind, batch, r, channels, groups, act, dtype='fp32', **more):
    return dict(kind=kind, batch=batch, r=r, channels=channels, groups=groups, act=act, dtype=dtype, **more)


def listed():
    return [
        # one field on its attention grid, the interactive use: latency
        dict(_norm('norm', 1, 43, 128, 32, 'silu'), name='norm_b1_r43_c128'),
        # the down-scaler's first convolution of 42 channels, seven to a group, in half precision: rows of 84 bytes
        dict(_norm('norm', 8, 211, 42, 6, 'relu', 'bf16'), name='norm_b8_r211_c42_bf16'),
        # the up-scaler's convolution on the middle grid at the throughput batch, the largest
        dict(_norm('norm', 64, 106, 128, 8, 'silu'), name='norm_b64_r106_c128'),
        # a training step at the reference's training batch
        dict(_norm('norm_train', 4, 71, 128, 32, 'silu', bits=32), name='norm_train_b4_r71'),
        # the same with the input kept in 8 bits, at four times the batch on the throughput benchmark's grid
        dict(_norm('norm_train', 16, 106, 128, 8, 'silu', bits=8), name='norm_train8_b16_r106'),
        # mixed precision: 211 x 211 nodes, 44 channels (the down-scaler's third convolution)
        dict(_norm('norm_train', 8, 211, 44, 4, 'silu', 'bf16', bits=8), name='norm_train8_b8_r211_c44_bf16'),
        # a checkpoint written and read back: the hidden values of one feed-forward block at the training batch ...
        dict(kind='checkpoint', rows=4 * 1849, width=256, dtype='fp32', name='checkpoint_b4_n1849'),
        # ... and in half precision at the throughput batch
        dict(kind='checkpoint', rows=64 * 2809, width=256, dtype='bf16', name='checkpoint_b64_n2809_bf16'),
        # an activation that keeps its input in 8 bits, forward and backward: one sample, and the throughput batch
        dict(kind='activation', rows=1849, width=256, act='relu', dtype='bf16', name='activation_b1_n1849_bf16'),
        dict(kind='activation', rows=64 * 2809, width=256, act='silu', dtype='fp32', name='activation_b64_n2809'),
        # weight gradients from an input in 8 bits: the output projection of the attention (four heads of 34) in mixed precision at the
        # training batch, and the feed-forward block's second layer at the throughput batch
        dict(kind='weight', rows=4 * 1849, outputs=128, inputs=136, dtype='bf16', name='weight_b4_n1849_128x136_bf16'),
        dict(kind='weight', rows=64 * 2809, outputs=128, inputs=256, dtype='fp32', name='weight_b64_n2809_128x256'),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['norm', 'norm', 'norm_train', 'norm_train', 'checkpoint', 'activation', 'weight', 'weight'])
    dtype = rng.choice(['fp32', 'fp32', 'bf16', 'fp16'])
    if kind in ('norm', 'norm_train'):
        channels = rng.choice([_log(rng, 8, 512), 8 * _log(rng, 1, 48)])
        groups = rng.choice([g for g in range(1, channels + 1) if channels % g == 0])
        r = _log(rng, 8, 421)
        most = 64 * 106 * 106 * 128 if kind == 'norm' else 16 * 106 * 106 * 128
        batch = _log(rng, 1, max(1, min(64, most // (r * r * channels))))
        while batch * r * r * channels > most:
            r -= 1
        if kind == 'norm':
            return _norm(kind, batch, r, channels, groups, rng.choice(['none', 'relu', 'silu']), dtype)
        # (a derivative with a kink would say on which side of it the last bit falls, so the steps are drawn without ReLU)
        return _norm(kind, batch, r, channels, groups, rng.choice(['none', 'silu', 'silu']), dtype, bits=rng.choice([8, 32]))
    rows = _log(rng, 1 if kind != 'weight' else 64, 64 * 2809)
    if kind == 'weight':
        # any widths: those of the model's layers and others
        outputs, inputs = (rng.choice([32, 128, 136, 256, _log(rng, 8, 256)]) for _ in range(2))
        while outputs * inputs > 128 * 256:
            outputs = max(8, outputs // 2)
        return dict(kind=kind, rows=rows, outputs=outputs, inputs=inputs, dtype=dtype)
    width = rng.choice([128, 136, 256, _log(rng, 8, 256)])
    if kind == 'checkpoint':
        return dict(kind=kind, rows=rows, width=width, dtype=dtype)
    return dict(kind=kind, rows=rows, width=width, act=rng.choice(['relu', 'silu']), dtype=dtype)


# ------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------
def _features(g, n, channels):
    """[n, channels] values as a layer of the model produces them: every channel with a mean and a spread of its own."""
    mean = torch.randn(channels, device='cuda', generator=g)
    spread = torch.exp(0.5 * torch.randn(channels, device='cuda', generator=g))
    return torch.randn(n, channels, device='cuda', generator=g) * spread + mean


def prepare(case, seed):
    g = torch.Generator('cuda').manual_seed(seed)
    dtype = TYPES[case['dtype']]
    state = {'case': case}
    if case['kind'] in ('norm', 'norm_train'):
        N, r, C = case['batch'], case['r'], case['channels']
        state['x'] = _features(g, N * r * r, C).view(N, r, r, C).to(dtype)
        state['w'] = 1.0 + 0.2 * torch.randn(C, device='cuda', generator=g)
        state['b'] = 0.2 * torch.randn(C, device='cuda', generator=g)
        if case['kind'] == 'norm_train':
            state['dy'] = torch.randn(N, r, r, C, device='cuda', generator=g).to(dtype)
        return state
    if case['kind'] == 'weight':
        # what a program has in hand in the backward pass: the checkpoint that the forward pass left, and the gradient
        x = _features(g, case['rows'], case['inputs']).to(dtype)
        state['codes'], state['steps'] = _codes(x)
        state['dy'] = torch.randn(case['rows'], case['outputs'], device='cuda', generator=g).to(dtype)
        return state
    state['x'] = _features(g, case['rows'], case['width']).to(dtype)
    if case['kind'] == 'activation':
        state['dy'] = torch.randn(case['rows'], case['width'], device='cuda', generator=g).to(dtype)
    return state


# ------------------------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------------------------
def _codes(x):
    """(codes [n], exponents of the steps [ceil(n / 32)]) of a checkpoint.  The step is the power of two 2^(E - 127) below which 127.5
    steps no longer exceed the block's largest magnitude, so x / step is exact and its rounding the same everywhere."""
    flat = x.reshape(-1).float()
    n = flat.numel()
    blocks = torch.nn.functional.pad(flat, (0, -n % BLOCK)).view(-1, BLOCK)
    bits = blocks.abs().amax(1).view(torch.int32)
    e = (((bits + 0x10000) >> 23) - 6).clamp_min(1)
    inverse = ((254 - e) << 23).view(torch.float32)
    q = torch.round(blocks * inverse[:, None]).to(torch.int8)
    return q.view(-1)[:n].contiguous(), e.to(torch.uint8)


def _values(codes, steps, shape):
    step = (steps.to(torch.int32) << 23).view(torch.float32)
    n = codes.numel()
    blocks = torch.nn.functional.pad(codes, (0, -n % BLOCK)).view(-1, BLOCK)
    return (blocks.float() * step[:, None]).view(-1)[:n].view(shape)


def _act(z, act):
    return z / (1.0 + torch.exp(-z)) if act == 'silu' else z.clamp_min(0) if act == 'relu' else z


def _dact(z, act):
    if act == 'silu':
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return (z > 0).to(z.dtype) if act == 'relu' else torch.ones_like(z)


def _plain_norm(state, train):
    case, x = state['case'], state['x']
    N, r, C, G = case['batch'], case['r'], case['channels'], case['groups']
    v = x.float().view(N, r * r, G, C // G)
    w, b = state['w'].view(1, 1, G, C // G), state['b'].view(1, 1, G, C // G)
    mean = v.mean((1, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt((v - mean).square().mean((1, 3), keepdim=True) + 1e-5)
    y = _act((v - mean) * rstd * w + b, case['act']).to(x.dtype).view(x.shape)
    if not train:
        return y
    if case['bits'] == 8:
        v = _values(*_codes(x), v.shape)
    xh = (v - mean) * rstd
    dz = state['dy'].float().view(v.shape) * _dact(xh * w + b, case['act'])
    dw, db = (dz * xh).sum((0, 1)).view(C), dz.sum((0, 1)).view(C)
    dz = dz * w
    c1, c2 = dz.mean((1, 3), keepdim=True), (dz * xh).mean((1, 3), keepdim=True)
    dx = (rstd * (dz - c1 - xh * c2)).to(x.dtype).view(x.shape)
    return y, dx, dw, db


def _plain(state):
    case = state['case']
    if case['kind'] in ('norm', 'norm_train'):
        return _plain_norm(state, case['kind'] == 'norm_train')
    if case['kind'] == 'weight':
        dy = state['dy'].float()
        return dy.t() @ _values(state['codes'], state['steps'], (case['rows'], case['inputs'])), dy.sum(0)
    x = state['x']
    kept = _values(*_codes(x), x.shape)
    if case['kind'] == 'checkpoint':
        return kept.to(x.dtype)
    return _act(x.float(), case['act']).to(x.dtype), (state['dy'].float() * _dact(kept, case['act'])).to(x.dtype)


# ------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ------------------------------------------------------------------------------------------------------------------
def _own(state):
    from spgt_b200 import ops
    from spgt_b200.extension.bind.checkpoint8 import activation8
    from spgt_b200.extension.bind.normalization import group_norm_act
    case = state['case']
    if case['kind'] == 'norm':
        with torch.no_grad():
            return group_norm_act(state['x'], case['groups'], state['w'], state['b'], 1e-5, case['act'])
    if case['kind'] == 'norm_train':
        x, w, b = (state[k].detach().requires_grad_() for k in ('x', 'w', 'b'))
        y = group_norm_act(x, case['groups'], w, b, 1e-5, case['act'], activation_bits=case['bits'])
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), state['dy']))
    if case['kind'] == 'checkpoint':
        return ops.restore8(ops.compress8(state['x']))
    if case['kind'] == 'activation':
        x = state['x'].detach().requires_grad_()
        y = activation8(x, case['act'])
        return y.detach(), torch.autograd.grad(y, x, state['dy'])[0]
    kept = ops.Checkpoint8(state['codes'], state['steps'], (case['rows'], case['inputs']), TYPES[case['dtype']])
    return ops.weight_gradient8(state['dy'], kept)


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------------------
# bytes and operations, results in 64 bits
# ------------------------------------------------------------------------------------------------------------------
def work(case):
    e, kept = BYTES[case['dtype']], 1 + 1 / BLOCK
    if case['kind'] in ('norm', 'norm_train'):
        n, C = case['batch'] * case['r'] ** 2 * case['channels'], case['channels']
        if case['kind'] == 'norm':                       # x in, y out
            return {'bytes': int(2 * n * e + 8 * C), 'flops': 10 * n}
        # forward x in, y out; backward dy and what is kept of x in, dx out.  A checkpoint is written as well.
        saved = 2 * kept * n if case['bits'] == 8 else e * n
        return {'bytes': int(4 * n * e + saved + 24 * C), 'flops': 40 * n}
    if case['kind'] == 'weight':
        rows, N, K = case['rows'], case['outputs'], case['inputs']
        return {'bytes': int(rows * (N * e + K * kept) + 4 * N * (K + 1)), 'flops': 2 * rows * N * K}
    n = case['rows'] * case['width']
    if case['kind'] == 'checkpoint':                     # x in, checkpoint out; checkpoint in, values out
        return {'bytes': int(2 * n * (e + kept)), 'flops': 3 * n}
    return {'bytes': int(n * (4 * e + 2 * kept)), 'flops': 25 * n}


def _kept64(x):
    """What a checkpoint of x stands for: the smallest step 2^e, e >= -126, of which the block's largest magnitude is less than 127.5."""
    flat = x.reshape(-1).double()
    rows = torch.zeros(-(-flat.numel() // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    rows[:flat.numel()] = flat
    rows = rows.reshape(-1, BLOCK)
    _, e = torch.frexp(rows.abs().max(dim=1, keepdim=True).values / 127.5)
    step = torch.ldexp(torch.ones_like(rows[:, :1]), e.clamp(min=-126))
    return (torch.round(rows / step) * step).reshape(-1)[:flat.numel()].reshape(x.shape)


def exact(case, seed):
    state = prepare(case, seed)
    act, sigmoid = case.get('act'), torch.sigmoid
    if case['kind'] == 'weight':
        e = state['steps'].double() - 127
        step = torch.exp2(e).repeat_interleave(BLOCK)[:state['codes'].numel()]
        x = (state['codes'].double() * step).reshape(case['rows'], case['inputs'])
        dy = state['dy'].double()
        return torch.einsum('rn,rk->nk', dy, x), torch.einsum('rn->n', dy)
    x = state['x'].double()
    slope = lambda z: sigmoid(z) * (1 + z * sigmoid(-z)) if act == 'silu' else (z > 0).double() if act == 'relu' else torch.ones_like(z)
    value = lambda z: z * sigmoid(z) if act == 'silu' else torch.relu(z) if act == 'relu' else z
    if case['kind'] == 'checkpoint':
        return _kept64(state['x'])
    if case['kind'] == 'activation':
        return value(x), state['dy'].double() * slope(_kept64(state['x']))
    N, C, G = case['batch'], case['channels'], case['groups']
    spread = lambda t: t.repeat_interleave(C // G, dim=1)[:, None, None, :]          # [N, G] -> [N, 1, 1, C]
    grouped = lambda t: t.reshape(N, -1, G, C // G).permute(0, 2, 1, 3).reshape(N, G, -1).mean(2)
    w, b = state['w'].double(), state['b'].double()
    mean = spread(grouped(x))
    r = spread((grouped((x - mean) ** 2) + 1e-5) ** -0.5)
    y = value((x - mean) * r * w + b)
    if case['kind'] == 'norm':
        return y
    xh = ((_kept64(state['x']) if case['bits'] == 8 else x) - mean) * r
    dz = state['dy'].double() * slope(xh * w + b)
    dx = r * (w * dz - spread(grouped(w * dz)) - xh * spread(grouped(w * dz * xh)))
    return y, dx, torch.einsum('nijc,nijc->c', dz, xh), torch.einsum('nijc->c', dz)
