"""Group normalisation with an activation, channels last, and activation checkpoints in 8 bits, against plain implementations in
64 bits.  U = 2^-24 is the relative error of one fp32 rounding; a sum in fixed order over chains of at most 64 terms, their merges and
five shuffles is off by at most 96 U of the sum of magnitudes, a sigmoid from the hardware exponential by 32 U."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _rand(*shape, seed=0, dtype=torch.float32, scale=1.0, mean=0.0):
    g = torch.Generator('cuda').manual_seed(seed)
    return (torch.randn(*shape, device='cuda', generator=g) * scale + mean).to(dtype)


def _rounded(t, dtype):
    """Half a step of a stored result of this size."""
    return 0.0 if dtype == torch.float32 else t.abs() * (torch.finfo(dtype).eps / 2) + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def _within(got, want, tol):
    """Every value within its tolerance; NaN exactly where expected."""
    got = got.double()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan())
    bad = ((got - want).abs() > tol) & ~want.isnan() & (got != want)
    assert not bad.any(), (int(bad.sum()), got[bad][:4].tolist(), want[bad][:4].tolist(), (tol + 0 * want)[bad][:4].tolist())


def _steps64(x):
    """(codes, step exponents E) of a checkpoint from its definition."""
    flat = x.reshape(-1).double()
    blocks = torch.nn.functional.pad(flat, (0, -flat.numel() % 32)).view(-1, 32)
    amax = blocks.abs().amax(1)
    _, e = torch.frexp(amax / 127.5)
    e = torch.where(amax == 0, torch.full_like(e, -126), e.clamp_min(-126))      # (the smallest step does for zeros)
    finite = blocks.isfinite().all(1)
    q = torch.round(blocks / torch.exp2(e.double())[:, None])
    q = torch.where(finite[:, None], q, torch.zeros_like(q))
    q = torch.where((e == 122)[:, None], q.clamp(-63, 63), q)                     # (64 steps of 2^122 are no finite fp32 number)
    return q.view(-1)[:flat.numel()].to(torch.int8), torch.where(finite, e + 127, torch.full_like(e, 255)).to(torch.uint8)


def _kept64(x):
    q, e = _steps64(x)
    step = torch.where(e == 255, torch.full_like(e, 1, dtype=torch.float64) * float('nan'), torch.exp2(e.double() - 127))
    return (q.double() * step.repeat_interleave(32)[:q.numel()]).view(x.shape)


def _act64(z, act):
    if act in (None, 'none'):
        return z
    if act == 'relu':
        return torch.relu(z)
    y = z * torch.sigmoid(z)
    return y * torch.sigmoid(y) if act == 'silu2' else y


def _slope64(z, act):
    if act in (None, 'none'):
        return torch.ones_like(z)
    if act == 'relu':
        return (z > 0).double()
    silu = lambda t: torch.sigmoid(t) * (1 + t * torch.sigmoid(-t))
    return silu(z * torch.sigmoid(z)) * silu(z) if act == 'silu2' else silu(z)


# ---------------------------------------------------------------------------------------------------------------------------------
# checkpoints
# ---------------------------------------------------------------------------------------------------------------------------------
def _awkward(n, dtype):
    x = _rand(n, seed=n, dtype=torch.float32) * torch.exp(3 * _rand(n, seed=n + 1))
    if n > 40:
        x[32:64] = 0                                           # a block of zeros
        x[7] = 127.5 * 4                                       # the step's border, and just below it
        x[70 % n] = 127.4375
    return x.to(dtype)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n', [0, 1, 3, 31, 32, 33, 100, 1023, 8 * 1024, 50001])
def test_checkpoint_codes_are_the_definition(dtype, n):
    from spgt_b200 import ops
    x = _awkward(n, dtype)
    kept = ops.compress8(x)
    q, e = _steps64(x)
    assert torch.equal(kept.codes, q) and torch.equal(kept.steps, e)
    assert kept.nbytes() == n + (n + 31) // 32
    back = kept.restore()
    want = _kept64(x)
    if dtype == torch.float16:
        want = want.clamp(-65504, 65504)
    assert back.dtype == dtype and torch.equal(back.isnan(), want.isnan()) and torch.equal(back.nan_to_num(0), want.to(dtype).nan_to_num(0))


def test_checkpoint_extremes():
    from spgt_b200 import ops
    x = torch.zeros(7 * 32, device='cuda')
    x[0] = 3.4028234e38; x[1] = 1.0                            # the largest number
    x[32] = 1.0e-45; x[33] = 1.1754944e-38; x[34] = -3.0e-39   # subnormal ones
    x[64] = float('inf'); x[65] = 2.0
    x[96] = float('nan'); x[97] = -2.0
    x[128] = float('-inf')
    x[160:192] = 1.9921875 * 2.0 ** torch.arange(-16., 16., device='cuda')
    x[192] = -0.0
    kept = ops.compress8(x)
    q, e = _steps64(x)
    assert torch.equal(kept.codes, q) and torch.equal(kept.steps, e)
    back = kept.restore()
    assert torch.equal(back.isnan(), _kept64(x).isnan()) and int(back.isnan().sum()) == 96
    half = torch.tensor([65504.0, -65504.0, 1.0], device='cuda', dtype=torch.float16)
    assert torch.equal(ops.compress8(half).restore()[:2], half[:2])     # 64 steps of 1024 would be an infinity in fp16
    back = ops.compress8(x.nan_to_num(0, 0, 0)).restore()
    step = torch.exp2(ops.compress8(x.nan_to_num(0, 0, 0)).steps.double() - 127).repeat_interleave(32)
    assert ((back.double() - x.nan_to_num(0, 0, 0).double()).abs() <= step / 2)[1:].all() and back[0] == 63 * 2.0 ** 122


@pytest.mark.parametrize('act', [None, 'relu', 'silu', 'silu2'])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', [(1,), (3, 5), (1849, 256), (0, 4), (7, 11, 13)])
def test_activation8(act, dtype, shape):
    from spgt_b200.extension.bind.checkpoint8 import activation8
    x = _rand(*shape, seed=1, dtype=dtype, scale=3.0).requires_grad_()
    dy = _rand(*shape, seed=2, dtype=dtype)
    y = activation8(x, act)
    want = _act64(x.detach().double(), act)
    _within(y.detach(), want, 64 * U * (want.abs() + x.detach().double().abs()) + _rounded(want, dtype))
    dx, = torch.autograd.grad(y, x, dy)
    want = dy.double() * _slope64(_kept64(x.detach()), act)
    _within(dx, want, 128 * U * dy.double().abs() * (1 + _kept64(x.detach()).abs()) + _rounded(want, dtype))
    with torch.no_grad():
        assert torch.equal(activation8(x, act), y)


def test_activation8_not_finite():
    from spgt_b200 import ops
    x = torch.ones(96, device='cuda')
    x[3], x[40], x[41] = float('nan'), float('inf'), -200.0
    for act in ('relu', 'silu', 'silu2', None):
        y, kept = ops.activation8(x, act)
        assert y[3].isnan() and y[40] == float('inf') and torch.equal(y[64:], y[64:65].expand(32))
        dx = ops.activation8_backward(torch.ones(96, device='cuda'), kept, act)
        assert (act is None or dx[:64].isnan().all()) and dx[64:].isfinite().all()


# ---------------------------------------------------------------------------------------------------------------------------------
# group normalisation
# ---------------------------------------------------------------------------------------------------------------------------------
def _norm64(x, G, w, b, eps, act, dy=None, kept=None):
    """Values and tolerances from the definition: {'y', 'dx', 'dw', 'db'} -> (value, tolerance)."""
    N, C = x.shape[0], x.shape[-1]
    v = x.double().reshape(N, -1, G, C // G)
    one, zero = torch.ones(C, device=x.device, dtype=torch.float64), torch.zeros(C, device=x.device, dtype=torch.float64)
    w, b = (one if w is None else w.double()).view(G, -1), (zero if b is None else b.double()).view(G, -1)
    mean = v.mean((1, 3), keepdim=True)
    var = (v - mean).square().mean((1, 3), keepdim=True)
    r = (var + eps).rsqrt()
    big = v.abs().amax((1, 3), keepdim=True)
    # the mean is off by 96 U of the magnitudes, which the variance feels in second order and through its own sum
    e_mean = 96 * U * big
    e_r = r * (100 * U + 0.5 * (e_mean * r) ** 2)

    def at(u):
        xh = (u - mean) * r
        return xh, e_mean * r + (u - mean).abs() * e_r + 4 * U * xh.abs()
    xh, e_xh = at(v)
    z, e_z = xh * w + b, e_xh * w.abs() + 4 * U * ((xh * w).abs() + b.abs())
    out = {'y': (_act64(z, act), 1.21 * e_z + 64 * U * z.abs())}
    if dy is not None:
        d = dy.double().reshape(v.shape)
        if kept is not None:
            xh, e_xh = at(kept.reshape(v.shape))
        z, e_z = xh * w + b, e_xh * w.abs() + 4 * U * ((xh * w).abs() + b.abs())
        dz = d * _slope64(z, act)
        if act == 'relu':                                      # the last bit says on which side of the kink a value lies
            e_dz = d.abs() * (z.abs() <= e_z)
        else:
            e_dz = d.abs() * (0.0 if act in (None, 'none') else 1.0) * (1.2 * e_z + 128 * U * (1 + z.abs()))
        t, s = w * dz, lambda q: q.mean((1, 3), keepdim=True)
        c1, c2 = s(t), s(t * xh)
        e_t = w.abs() * e_dz + 4 * U * t.abs()
        e_c1 = s(e_t) + 100 * U * s(t.abs())
        e_c2 = s(e_t * xh.abs() + t.abs() * e_xh) + 100 * U * s((t * xh).abs())
        inner = t - c1 - xh * c2
        out['dx'] = (r * inner, r * (e_t + e_c1 + e_xh * c2.abs() + xh.abs() * e_c2 + 8 * U * (t.abs() + c1.abs() + (xh * c2).abs())) + e_r * inner.abs())
        out['db'] = (dz.sum((0, 1)).view(C), (e_dz.sum((0, 1)) + 100 * U * dz.abs().sum((0, 1))).view(C))
        out['dw'] = ((dz * xh).sum((0, 1)).view(C), ((e_dz * xh.abs() + dz.abs() * e_xh).sum((0, 1)) + 100 * U * (dz * xh).abs().sum((0, 1))).view(C))
    return {k: (a, e) if k in ('dw', 'db') else (a.reshape(x.shape), e.expand_as(a).reshape(x.shape)) for k, (a, e) in out.items()}


SHAPES = [
    # N, pixels, C, G
    (1, (1,), 1, 1), (2, (3, 5), 1, 1), (5, (1,), 64, 4), (2, (5,), 7, 7), (3, (7, 7), 42, 6), (3, (11, 13), 33, 3), (2, (2, 3, 5), 10, 2),
    (1, (29, 29), 128, 32), (2, (43, 43), 128, 8), (4, (53,), 44, 4), (2, (9, 9), 512, 1), (2, (9, 9), 511, 73), (1, (6,), 2048, 16), (300, (2, 2), 32, 8),
    (2, (97, 101), 96, 96), (1, (421, 421), 6, 3),
]


@pytest.mark.parametrize('N,pixels,C,G', SHAPES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('act', [None, 'relu', 'silu', 'silu2'])
def test_group_norm(N, pixels, C, G, dtype, act):
    from spgt_b200.extension.bind.normalization import group_norm_act
    x = _rand(N, *pixels, C, seed=C, dtype=dtype, scale=1.5, mean=0.7).requires_grad_()
    w, b = _rand(C, seed=1, scale=0.3, mean=1.0).requires_grad_(), _rand(C, seed=2, scale=0.3).requires_grad_()
    dy = _rand(N, *pixels, C, seed=3, dtype=dtype)
    x64 = x.detach()
    for bits in (32, 8):
        want = _norm64(x64, G, w.detach(), b.detach(), 1e-5, act, dy, _kept64(x64) if bits == 8 else None)
        y = group_norm_act(x, G, w, b, 1e-5, act, activation_bits=bits)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
        for k, got in (('y', y.detach()), ('dx', dx), ('dw', dw), ('db', db)):
            value, tol = want[k]
            _within(got, value, tol + (_rounded(value, dtype) if k in ('y', 'dx') else 0.0))
    with torch.no_grad():
        assert torch.equal(group_norm_act(x, G, w, b, 1e-5, act), y)


@pytest.mark.parametrize('dtype', TYPES)
def test_group_norm_4096_channels(dtype):
    from spgt_b200 import ops
    C = 2048 if dtype == torch.float32 else 4096
    x, dy = _rand(2, 3, C, seed=1, dtype=dtype), _rand(2, 3, C, seed=2, dtype=dtype)
    for G in (1, 4, C // 2, C):
        want = _norm64(x, G, None, None, 1e-3, 'silu', dy)
        y, stats, _ = ops.group_norm(x, G, None, None, 1e-3, 'silu')
        dx, dw, db = ops.group_norm_backward(dy, x, G, None, None, stats, 'silu')
        for k, got in (('y', y), ('dx', dx), ('dw', dw), ('db', db)):
            _within(got, want[k][0], want[k][1] + (_rounded(want[k][0], dtype) if k in ('y', 'dx') else 0.0))


@pytest.mark.parametrize('mean,scale', [(1000.0, 1.0), (-3.0e4, 0.5), (0.0, 1e-12), (0.0, 1e12)])
def test_group_norm_far_means_and_scales(mean, scale):
    """The corner pixel is zero, as on a Dirichlet frame: no value of the data may serve as the others' origin."""
    from spgt_b200 import ops
    x = _rand(2, 31, 33, 48, seed=5, scale=scale, mean=mean)
    x[:, 0, :] = 0
    dy = _rand(2, 31, 33, 48, seed=6)
    w, b = _rand(48, seed=1, scale=0.3, mean=1.0), _rand(48, seed=2)
    want = _norm64(x, 6, w, b, 1e-5, 'silu', dy)
    y, stats, _ = ops.group_norm(x, 6, w, b, 1e-5, 'silu')
    dx, dw, db = ops.group_norm_backward(dy, x, 6, w, b, stats, 'silu')
    for k, got in (('y', y), ('dx', dx), ('dw', dw), ('db', db)):
        _within(got, *want[k])


def test_group_norm_constant_and_not_finite():
    from spgt_b200 import ops
    x = torch.full((3, 5, 7, 16), 3.25, device='cuda')
    b = _rand(16, seed=2)
    y, stats, _ = ops.group_norm(x, 4, None, b, 1e-5, None)
    assert torch.equal(y, b.expand_as(y)) and torch.equal(stats[..., 0], torch.full_like(stats[..., 0], 3.25))
    x = _rand(3, 5, 7, 16, seed=1)
    clean, clean_stats, _ = ops.group_norm(x, 4, None, b, 1e-5, 'relu')
    x[1, 2, 3, 5] = float('nan')
    x[2, 0, 0, 15] = float('inf')
    y, stats, kept = ops.group_norm(x, 4, None, b, 1e-5, 'relu', compress=True)
    hit = torch.zeros(3, 4, dtype=torch.bool, device='cuda')
    hit[1, 1] = hit[2, 3] = True
    mask = hit.repeat_interleave(4, 1)[:, None, None, :].expand_as(y)
    assert torch.equal(y.isnan(), mask) and torch.equal(y[~mask], clean[~mask])       # the other groups as without it
    dx, dw, db = ops.group_norm_backward(torch.ones_like(x), x, 4, None, b, stats, 'relu')
    assert dx[mask].isnan().all() and dx[~mask].isfinite().all()


@pytest.mark.parametrize('dtype', TYPES)
def test_unaligned_views_and_empty(dtype):
    from spgt_b200 import ops
    n = 3 * 5 * 7 * 12
    flat, w = _rand(n + 1, seed=1, dtype=dtype), _rand(13, seed=2)
    x = flat[1:].view(3, 5, 7, 12)
    for a, c in zip(ops.group_norm(x, 3, w[1:], None)[:2], ops.group_norm(x.clone(), 3, w[1:].clone(), None)[:2]):
        assert torch.equal(a, c)
    assert torch.equal(ops.compress8(x).codes, ops.compress8(x.clone()).codes)
    dy = _rand(n + 1, seed=3, dtype=dtype)[1:].view_as(x)
    stats = ops.group_norm(x.clone(), 3, None, None)[1]
    for a, c in zip(ops.group_norm_backward(dy, x, 3, None, None, stats), ops.group_norm_backward(dy.clone(), x.clone(), 3, None, None, stats)):
        assert torch.equal(a, c)
    for a, c in zip(ops.weight_gradient8(dy.view(-1, 12), ops.compress8(x.reshape(-1, 12))), ops.weight_gradient8(dy.clone().view(-1, 12), ops.compress8(x.clone().reshape(-1, 12)))):
        assert torch.equal(a, c)
    for shape in ((0, 5, 12), (2, 0, 12)):
        x = torch.empty(shape, device='cuda', dtype=dtype)
        y, stats, kept = ops.group_norm(x, 3, None, None, compress=True)
        assert y.shape == shape and kept.nbytes() == 0
        dx, dw, db = ops.group_norm_backward(x, kept, 3, None, None, stats)
        assert dx.shape == shape and not dw.any() and not db.any()


@pytest.mark.parametrize('N,P,C,G', [(3, 35, 7, 1), (5, 900, 64, 8)])
def test_group_norm_in_place(N, P, C, G):
    """The C entry point takes y = x, without and with a checkpoint of x."""
    from spgt_b200._lib import lib
    from spgt_b200 import ops
    x = _rand(N, P, C, seed=1)
    want, stats, kept = ops.group_norm(x, G, None, None, 1e-5, 'silu', compress=True)
    need = lib.spgt_group_norm_workspace_bytes(N, P, C, G, 0)
    for compress in (False, True):
        y, s = x.clone(), torch.empty_like(stats)
        codes, steps = torch.empty_like(kept.codes), torch.empty_like(kept.steps)
        ws = torch.empty(need, dtype=torch.uint8, device='cuda')
        rc = lib.spgt_group_norm_fwd(y.data_ptr(), None, None, y.data_ptr(), s.data_ptr(), codes.data_ptr() if compress else None, steps.data_ptr() if compress else None,
                                     N, P, C, G, 1e-5, 2, 0, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and torch.equal(y, want) and torch.equal(s, stats)
        assert not compress or (torch.equal(codes, kept.codes) and torch.equal(steps, kept.steps))


def test_group_norm_several_units():
    """More samples than one unit holds in either pass: as sample by sample."""
    from spgt_b200 import ops
    N, P, C, G = 9, 180 * 180, 128, 4                          # 16.6 MB a sample
    x, dy = _rand(N, P, C, seed=1, mean=0.3), _rand(N, P, C, seed=2)
    w, b = _rand(C, seed=3, mean=1.0, scale=0.2), _rand(C, seed=4)
    y, stats, kept = ops.group_norm(x, G, w, b, 1e-5, 'silu', compress=True)
    dx, dw, db = ops.group_norm_backward(dy, x, G, w, b, stats, 'silu')
    dx8, dw8, db8 = ops.group_norm_backward(dy, kept, G, w, b, stats, 'silu')
    sums = [torch.zeros(C, device='cuda', dtype=torch.float64) for _ in range(4)]
    for n in range(N):
        want = _norm64(x[n:n + 1], G, w, b, 1e-5, 'silu', dy[n:n + 1])
        _within(y[n:n + 1], *want['y'])
        _within(dx[n:n + 1], *want['dx'])
        want8 = _norm64(x[n:n + 1], G, w, b, 1e-5, 'silu', dy[n:n + 1], _kept64(x[n:n + 1]))
        _within(dx8[n:n + 1], *want8['dx'])
        for s, v in zip(sums, (want['dw'][0], want['db'][0], want8['dw'][0], want8['db'][0])):
            s += v
    for got, want in zip((dw, db, dw8, db8), sums):
        assert float((got.double() - want).norm() / want.norm()) < 2e-6


def test_group_norm_in_place_buffers_are_kept():
    """Nothing is written behind the outputs, whatever part of a vector they end in."""
    from spgt_b200._lib import lib
    from spgt_b200 import ops
    for N, P, C, G in ((2, 35, 7, 1), (3, 9, 42, 6), (1, 1, 3, 3)):
        n = N * P * C
        x, w = _rand(n, seed=1), _rand(C, seed=2)
        y = torch.full((n + 8,), 7.0, device='cuda')
        codes, steps = torch.full((n + 8,), 7, dtype=torch.int8, device='cuda'), torch.full(((n + 31) // 32 + 4,), 7, dtype=torch.uint8, device='cuda')
        stats = torch.full((N * G * 2 + 4,), 7.0, device='cuda')
        need = lib.spgt_group_norm_workspace_bytes(N, P, C, G, 0)
        ws = torch.empty(need, dtype=torch.uint8, device='cuda')
        rc = lib.spgt_group_norm_fwd(x.data_ptr(), w.data_ptr(), None, y.data_ptr(), stats.data_ptr(), codes.data_ptr(), steps.data_ptr(), N, P, C, G,
                                     1e-5, 0, 0, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert (y[n:] == 7).all() and (codes[n:] == 7).all() and (steps[(n + 31) // 32:] == 7).all() and (stats[N * G * 2:] == 7).all()
        assert torch.equal(y[:n].view(N, P, C), ops.group_norm(x.view(N, P, C), G, w, None)[0])


# ---------------------------------------------------------------------------------------------------------------------------------
# weight gradients
# ---------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,N,K', [(1, 1, 1), (7, 8, 16), (63, 32, 130), (65, 1, 128), (1849, 128, 136), (1849, 256, 128), (2809, 128, 256),
                                      (1000, 34, 42), (130, 300, 520), (4096, 33, 31), (20000, 128, 256), (517, 129, 257), (200000, 8, 16), (190001, 5, 130)])
def test_weight_gradient8(dtype, rows, N, K):
    from spgt_b200 import ops
    x, dy = _rand(rows, K, seed=1, dtype=dtype, mean=0.5), _rand(rows, N, seed=2, dtype=dtype)
    kept = ops.compress8(x)
    dw, db = ops.weight_gradient8(dy, kept)
    v, d = _kept64(x), dy.double()
    # products are exact in fp32; an accumulator takes at most 80 additions that truncate (2 U each) before its sum moves on, and the
    # sums of fewer than 64 pieces are added up in chains of at most 19
    _within(dw, d.t() @ v, 192 * U * (d.abs().t() @ v.abs()) + 1e-37)
    # a thread adds up at most rows / (148 * 16) values in a row, at most 64 of them are added in order, and at most 19 blocks' results
    _within(db, d.sum(0), (192 + rows / 2000) * U * d.abs().sum(0))
    again = ops.weight_gradient8(dy, kept, column_sums=False)
    assert torch.equal(again[0], dw) and again[1] is None


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows', [1, 31, 33, 63, 65, 129, 4765, 28421])
@pytest.mark.parametrize('N,K', [(8, 16), (128, 112), (40, 128), (128, 144), (120, 240), (128, 256)])
def test_weight_gradient8_one_tile(dtype, rows, N, K):
    """Widths of one tile, whose blocks are copied as they lie in memory where the steps start on a 16-byte boundary and piece by piece where
    they do not: the same result, and rows past the end count for nothing."""
    from spgt_b200 import ops
    x, dy = _rand(rows, K, seed=1, dtype=dtype, mean=0.5), _rand(rows, N, seed=2, dtype=dtype)
    kept = ops.compress8(x)
    dw, db = ops.weight_gradient8(dy, kept)
    v, d = _kept64(x), dy.double()
    _within(dw, d.t() @ v, 192 * U * (d.abs().t() @ v.abs()) + 1e-37)
    _within(db, d.sum(0), (192 + rows / 2000) * U * d.abs().sum(0))
    room = torch.empty(kept.steps.numel() + 1, device='cuda', dtype=torch.uint8)
    room[1:] = kept.steps
    dw1, db1 = ops.weight_gradient8(dy, ops.Checkpoint8(kept.codes, room[1:], x.shape, dtype))
    assert torch.equal(dw, dw1) and torch.equal(db, db1)
    # what lies behind the last row is not read into the sums
    more = torch.full((rows + 64, N), float('nan'), device='cuda', dtype=dtype)
    more[:rows] = dy
    codes = torch.cat((kept.codes.view(-1), torch.full((64 * K,), 127, device='cuda', dtype=torch.int8)))
    steps = torch.cat((kept.steps.view(-1), torch.full((64 * K // 32 + 1,), 255, device='cuda', dtype=torch.uint8)))
    dw2, db2 = ops.weight_gradient8(more[:rows], ops.Checkpoint8(codes[:rows * K], steps[:(rows * K + 31) // 32], x.shape, dtype))
    assert torch.equal(dw, dw2) and torch.equal(db, db2)


def test_weight_gradient8_no_rows():
    from spgt_b200 import ops
    dw, db = ops.weight_gradient8(torch.empty(0, 5, device='cuda'), ops.compress8(torch.empty(0, 9, device='cuda')))
    assert dw.shape == (5, 9) and not dw.any() and not db.any()


@pytest.mark.parametrize('dtype', TYPES)
def test_weight_gradient8_not_finite(dtype):
    """A NaN or an infinity reaches its own row or column and no other."""
    from spgt_b200 import ops
    x, dy = _rand(700, 64, seed=1, dtype=dtype), _rand(700, 40, seed=2, dtype=dtype)
    clean, _ = ops.weight_gradient8(dy, ops.compress8(x))
    dy[300, 7] = float('nan')
    dy[301, 9] = float('inf')
    x[650, 40] = float('nan')                                   # columns 32 .. 63 of that row
    dw, db = ops.weight_gradient8(dy, ops.compress8(x))
    assert dw[7].isnan().all() and not dw[9].isfinite().any() and dw[:, 32:].isnan().all()
    keep = torch.ones(40, dtype=torch.bool, device='cuda')
    keep[7] = keep[9] = False
    assert torch.equal(dw[keep][:, :32], clean[keep][:, :32])
    assert db[7].isnan() and db[9] == float('inf') and db[keep].isfinite().all()


@pytest.mark.parametrize('dtype', TYPES)
def test_linear8(dtype):
    from spgt_b200.extension.bind.checkpoint8 import linear8
    x, w, b = (_rand(*s, seed=i, dtype=dtype, scale=0.5).requires_grad_() for i, s in enumerate(((3, 50, 24), (40, 24), (40,))))
    dy = _rand(3, 50, 40, seed=9, dtype=dtype)
    y = linear8(x, w, b)
    assert torch.equal(y, torch.nn.functional.linear(x, w, b))
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert dx.dtype == dw.dtype == db.dtype == dtype
    d, v = dy.double().view(-1, 40), _kept64(x.detach()).view(-1, 24)
    _within(dw, d.t() @ v, 128 * U * (d.abs().t() @ v.abs()) + _rounded(d.t() @ v, dtype))
    _within(db, d.sum(0), 128 * U * d.abs().sum(0) + _rounded(d.sum(0), dtype))
    assert torch.equal(dx, torch.matmul(dy, w.detach()))
    only, = torch.autograd.grad(linear8(x, w.detach(), b.detach()), x, dy)
    assert torch.equal(only, dx)


# ---------------------------------------------------------------------------------------------------------------------------------
# as a program uses them
# ---------------------------------------------------------------------------------------------------------------------------------
def _block(x, w, b, lw, lb):
    """A normalised block and a dense layer that keep their inputs in 8 bits."""
    from spgt_b200.extension.bind.checkpoint8 import activation8, linear8
    from spgt_b200.extension.bind.normalization import group_norm_act
    h = group_norm_act(x, 4, w, b, 1e-5, 'silu', activation_bits=8)
    return activation8(linear8(h, lw, lb), 'silu')


def _block_inputs(seed=0):
    x, dy = _rand(2, 23, 23, 32, seed=seed), _rand(2, 23, 23, 48, seed=seed + 1)
    params = [_rand(32, seed=3, mean=1.0, scale=0.2), _rand(32, seed=4), _rand(48, 32, seed=5, scale=0.2), _rand(48, seed=6)]
    return x, dy, params


def _block_step(x, dy, params):
    leaves = [t.detach().requires_grad_() for t in (x, *params)]
    y = _block(*leaves)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


def test_a_run_of_them_and_again():
    """Gradients of a chain of the operators: the formulas' at the rounded inputs; the same bits every time."""
    x, dy, params = _block_inputs()
    got = _block_step(x, dy, params)
    for a, c in zip(got, _block_step(x, dy, params)):
        assert torch.equal(a, c)
    w, b, lw, lb = (p.double() for p in params)
    n = _norm64(x, 4, w, b, 1e-5, 'silu')['y'][0]
    pre = torch.nn.functional.linear(n, lw, lb)
    assert float((got[0] - _act64(pre, 'silu')).norm() / _act64(pre, 'silu').norm()) < 1e-6
    # (the roundings to 8 bits are of the kernel's own fp32 values: at 64 bits some would fall on the other side of a step)
    from spgt_b200 import ops
    h, stats, kept = ops.group_norm(x, 4, params[0], params[1], 1e-5, 'silu', compress=True)
    pre32 = torch.nn.functional.linear(h, params[2], params[3])
    dpre = dy.double() * _slope64(_kept64(pre32), 'silu')
    dlw = dpre.view(-1, 48).t() @ _kept64(h).view(-1, 32)
    dh = dpre @ lw
    want = _norm64(x, 4, params[0], params[1], 1e-5, 'silu', dh, _kept64(x))
    for a, c in zip(got[1:], (want['dx'][0], want['dw'][0], want['db'][0], dlw, dpre.view(-1, 48).sum(0))):
        assert float((a.double() - c).norm() / c.norm()) < 2e-6


def test_gradient_against_differences():
    """Directional derivative of the 32-bit operator by central differences in 64 bits."""
    from spgt_b200 import ops
    x, dy = _rand(2, 13, 13, 24, seed=1), _rand(2, 13, 13, 24, seed=2)
    w, b = _rand(24, seed=3, mean=1.0, scale=0.2), _rand(24, seed=4)
    y, stats, _ = ops.group_norm(x, 3, w, b, 1e-5, 'silu')
    grads = ops.group_norm_backward(dy, x, 3, w, b, stats, 'silu')
    dirs = [_rand(*t.shape, seed=7 + i).double() for i, t in enumerate((x, w, b))]
    f = lambda h: float((_norm64(x.double() + h * dirs[0], 3, w.double() + h * dirs[1], b.double() + h * dirs[2], 1e-5, 'silu')['y'][0] * dy.double()).sum())
    h = 1e-5
    slope = (f(h) - f(-h)) / (2 * h)
    assert abs(sum(float((g.double() * d).sum()) for g, d in zip(grads, dirs)) - slope) < 1e-5 * (abs(slope) + 1)


def test_streams_and_graphs():
    x, dy, params = _block_inputs()
    want = _block_step(x, dy, params)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _block_step(x, dy, params)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    # two captured graphs, replayed one after the other and at once on two streams, on other inputs than at capture
    graphs = []
    for k in range(2):
        bx, bdy, _ = _block_inputs(seed=50 + k)
        with torch.cuda.stream(side):
            _block_step(bx, bdy, params)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _block_step(bx, bdy, params)
        graphs.append((g, bx, bdy, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for repeat in range(3):
        wants = []
        for k, (g, bx, bdy, out) in enumerate(graphs):
            nx, ndy, _ = _block_inputs(seed=100 + 10 * repeat + k)
            bx.copy_(nx); bdy.copy_(ndy)
            wants.append(_block_step(nx, ndy, params))
        for s, (g, *_) in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for (g, bx, bdy, out), want in zip(graphs, wants):
            assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_refusals_on_device():
    from spgt_b200 import ops
    from spgt_b200.extension.bind.checkpoint8 import activation8, linear8
    from spgt_b200.extension.bind.normalization import group_norm_act
    x = _rand(2, 4, 4, 12, seed=1)
    kept = ops.compress8(x)
    bad = [
        (ValueError, lambda: ops.group_norm(x, 5, None, None)), (ValueError, lambda: ops.group_norm(x, 0, None, None)),
        (ValueError, lambda: ops.group_norm(x[0, 0, 0], 3, None, None)), (ValueError, lambda: ops.group_norm(x.transpose(1, 2), 3, None, None)),
        (TypeError, lambda: ops.group_norm(x.double(), 3, None, None)), (ValueError, lambda: ops.group_norm(x, 3, torch.ones(11, device='cuda'), None)),
        (TypeError, lambda: ops.group_norm(x, 3, torch.ones(12, device='cuda').half(), None)), (ValueError, lambda: ops.group_norm(x, 3, torch.ones(12), None)),
        (ValueError, lambda: ops.group_norm(x, 3, None, None, eps=-1.0)), (ValueError, lambda: ops.group_norm(x.new_empty(1, 2, 1000 * 3 + 1), 1, None, None)),
        (ValueError, lambda: group_norm_act(x, 3, activation_bits=4)),
        (ValueError, lambda: ops.group_norm_backward(x, x, 3, None, None, torch.ones(2, 4, 2, device='cuda'))),
        (ValueError, lambda: ops.group_norm_backward(x[:1], x, 3, None, None, torch.ones(2, 3, 2, device='cuda'))),
        (TypeError, lambda: ops.group_norm_backward(x.half(), x, 3, None, None, torch.ones(2, 3, 2, device='cuda'))),
        (ValueError, lambda: ops.Checkpoint8(kept.codes, kept.steps[:-1], x.shape)), (ValueError, lambda: ops.Checkpoint8(kept.codes, kept.steps, (5,))),
        (TypeError, lambda: ops.Checkpoint8(kept.codes, kept.steps, x.shape, torch.float64)), (TypeError, lambda: ops.Checkpoint8(kept.steps, kept.steps, x.shape)),
        (ValueError, lambda: ops.weight_gradient8(x[:1], kept)), (ValueError, lambda: ops.weight_gradient8(x.view(-1, 12), kept)),
        (ValueError, lambda: ops.activation8_backward(x[:1], kept, 'relu')), (TypeError, lambda: ops.compress8(x.long())),
    ]
    for error, call in bad:
        with pytest.raises(error):
            call()
    # a second derivative is refused, not wrong
    for f in (lambda t: group_norm_act(t, 3), lambda t: activation8(t, 'silu'), lambda t: linear8(t, torch.ones(5, 12, device='cuda'))):
        t = x.clone().requires_grad_()
        g, = torch.autograd.grad(f(t).square().sum(), t, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), t)


def test_calls_with_and_without_gradients_agree():
    """The same arguments are taken, and refused, whether or not a gradient is wanted."""
    from spgt_b200 import ops
    from spgt_b200.extension.bind.checkpoint8 import activation8, linear8
    from spgt_b200.extension.bind.normalization import group_norm_act
    x = _rand(2, 24, 9, 8, seed=1).permute(0, 2, 3, 1)          # not contiguous
    for f in (lambda t: group_norm_act(t, 4, None, None, 1e-5, 'silu'), lambda t: activation8(t, 'silu'),
              lambda t: linear8(t, torch.ones(3, 24, device='cuda'))):
        with torch.no_grad():
            want = f(x)
        assert torch.equal(f(x.clone(memory_format=torch.preserve_format).requires_grad_()).detach(), want)
        assert torch.equal(f(x.contiguous()), want)
    wide = ops.WEIGHT8_MOST + 1
    for w in (torch.ones(2, wide, device='cuda'), torch.ones(wide, 2, device='cuda')):
        with pytest.raises(ValueError):                         # before anything is kept for a backward pass that could not run
            linear8(torch.ones(3, w.shape[1], device='cuda', requires_grad=True), w)


def test_weight_gradient8_widest():
    from spgt_b200 import ops
    for N, K in ((ops.WEIGHT8_MOST, 40), (40, ops.WEIGHT8_MOST), (ops.WEIGHT8_MOST - 3, 33)):
        x, dy = _rand(67, K, seed=1), _rand(67, N, seed=2)
        kept = ops.compress8(x)
        dw, db = ops.weight_gradient8(dy, kept)
        v, d = _kept64(x), dy.double()
        _within(dw, d.t() @ v, 192 * U * (d.abs().t() @ v.abs()) + 1e-37)
        _within(db, d.sum(0), 192 * U * d.abs().sum(0))


@pytest.mark.parametrize('N,P,C,G', [(3000, 4, 8, 2), (1, 1, 2048, 64), (300, 1, 250, 5), (7, 2, 3, 3)])
def test_group_norm_backward_many_rows_of_sums(N, P, C, G):
    """Parameter gradients over many small samples and few or many channels."""
    from spgt_b200 import ops
    x, dy, w, b = _rand(N, P, C, seed=1), _rand(N, P, C, seed=2), _rand(C, seed=3), _rand(C, seed=4)
    y, stats, _ = ops.group_norm(x, G, w, b, 1e-3, None)
    dx, dw, db = ops.group_norm_backward(dy, x, G, w, b, stats, None)
    d, m, r = dy.double(), stats[..., 0].double(), stats[..., 1].double()
    xh = (x.double().view(N, P, G, -1) - m[:, None, :, None]) * r[:, None, :, None]
    xh = xh.reshape(N, P, C)
    # a sum of N P terms in chains of at most N / 128 + 64 + 12 additions, each term with the few roundings of xh
    n = N * P // 64 + 100
    _within(db, d.sum((0, 1)), n * U * d.abs().sum((0, 1)) + 1e-30)
    _within(dw, (d * xh).sum((0, 1)), n * U * (d * xh).abs().sum((0, 1)) + 1e-30)
    wd = (w.double() * d).view(N, P, G, -1)
    xg = xh.view(N, P, G, -1)
    want = r[:, None, :, None] * (wd - wd.mean((1, 3), keepdim=True) - xg * (wd * xg).mean((1, 3), keepdim=True))
    size = r[:, None, :, None] * (wd.abs() + wd.abs().mean((1, 3), keepdim=True) + xg.abs() * (wd * xg).abs().mean((1, 3), keepdim=True))
    _within(dx.view(N, P, G, -1), want, 100 * U * size + 1e-30)
