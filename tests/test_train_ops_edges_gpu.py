"""The training operators at the ends of their ranges: calls that their documentation allows or refuses."""
import pytest
import torch

from tests.helpers import rel_l2
from tests.test_train_ops_gpu import TYPES, U, _kept64, _norm64, _rand, _rounded, _within

pytestmark = pytest.mark.gpu


def test_statistics_of_no_pixels_are_zero():
    from spgt_b200 import ops
    for shape in ((2, 0, 12), (0, 5, 12)):
        dirt = [torch.full((128,), float('nan'), device='cuda') for _ in range(64)]     # what the next small allocation holds
        del dirt
        y, stats, _ = ops.group_norm(torch.empty(shape, device='cuda'), 3, None, None)
        assert y.shape == shape and stats.shape == (shape[0], 3, 2) and torch.equal(stats, torch.zeros_like(stats))


def test_unknown_activations_are_refused():
    """A name that the operators do not know is an error, with and without gradients, and not another activation."""
    from spgt_b200 import ops
    from spgt_b200.extension.bind.checkpoint8 import activation8
    from spgt_b200.extension.bind.normalization import group_norm_act
    x = _rand(2, 4, 4, 12, seed=1)
    leaf = x.clone().requires_grad_()
    kept = ops.compress8(x)
    stats = ops.group_norm(x, 3, None, None)[1]
    for name in ('gelu', 'tanh', 'ReLU', ''):
        for call in (lambda: group_norm_act(x, 3, activation=name), lambda: group_norm_act(leaf, 3, activation=name), lambda: activation8(x, name),
                     lambda: activation8(leaf, name), lambda: ops.group_norm(x, 3, None, None, act=name),
                     lambda: ops.group_norm_backward(x, x, 3, None, None, stats, name), lambda: ops.activation8(x, name),
                     lambda: ops.activation8_backward(x, kept, name)):
            with pytest.raises(ValueError, match='activation'):
                call()


def test_layers_follow_the_rule_of_the_configuration():
    """The model's layers take 'silu' as SiLU and any other name as ReLU, with the options as without."""
    from spgt_b200.network.layer import ConvResBlock2D, FeedForward
    torch.manual_seed(0)
    x = _rand(5, 40, seed=1).requires_grad_()
    image = _rand(2, 6, 9, 11, seed=2)
    for name in ('gelu', 'none', 'silu2', 'relu', 'silu'):
        ffn = FeedForward(40, 40, 64, 0.0, name).cuda()
        want = ffn.forward_train(x)
        ffn.activation_bits = 8
        assert rel_l2(ffn.forward_train(x), want) < 1e-5
    block = ConvResBlock2D(6, 24, 3, 1, 0.0, 'gelu', num_group=4).cuda()
    with torch.backends.cudnn.flags(allow_tf32=False):
        z = block.conv_layer(image)
        want = torch.relu(torch.nn.functional.group_norm(z, 4, block.norm.weight, block.norm.bias, 1e-5))
        assert rel_l2(block.forward_train(image), want) < 1e-5


def test_frozen_layer_keeps_no_checkpoint():
    from spgt_b200.extension.bind.checkpoint8 import linear8
    x, w, b = _rand(4096, 64, seed=1).requires_grad_(), _rand(32, 64, seed=2), _rand(32, seed=3)
    dy = _rand(4096, 32, seed=4)
    linear8(x, w, b)                                            # (the library's workspace is allocated once)
    before = torch.cuda.memory_allocated()
    y = linear8(x, w, b)
    assert torch.cuda.memory_allocated() - before == y.numel() * 4
    dx, = torch.autograd.grad(y, x, dy)
    assert torch.equal(dx, dy @ w)
    # only the bias, or only the weight
    lw, lb = w.clone().requires_grad_(), b.clone().requires_grad_()
    want_w, want_b = torch.autograd.grad(linear8(x.detach(), lw, lb), (lw, lb), dy)
    got, = torch.autograd.grad(linear8(x.detach(), w, lb), lb, dy)
    assert torch.equal(got, want_b)
    got, = torch.autograd.grad(linear8(x.detach(), lw, b), lw, dy)
    assert torch.equal(got, want_w)


@pytest.mark.parametrize('dims,dtype', [((8, 4100, 16), torch.float32), ((4100, 8, 16), torch.float32), ((8, 8, 4100), torch.float32), ((12, 20, 30), torch.float64)])
def test_feed_forward_that_linear8_does_not_take(dims, dtype):
    """Widths and types beyond linear8 train on the plain layers, as without the option."""
    from spgt_b200.network.layer import FeedForward
    torch.manual_seed(0)
    ffn = FeedForward(*dims, 0.0, 'silu').cuda().to(dtype)
    x, dy = _rand(6, dims[0], seed=1).to(dtype).requires_grad_(), _rand(6, dims[1], seed=2).to(dtype)

    def step():
        y = ffn.forward_train(x)
        return [y.detach(), *torch.autograd.grad(y, (x, *ffn.parameters()), dy)]
    want = step()
    ffn.activation_bits = 8
    assert all(torch.equal(a, c) for a, c in zip(step(), want))


def test_linear8_without_features():
    """A layer of no features in or out is refused before anything is kept for a backward pass that could not run."""
    from spgt_b200.extension.bind.checkpoint8 import linear8
    for K, N in ((0, 3), (3, 0)):
        with pytest.raises(ValueError):
            linear8(torch.ones(5, K, device='cuda', requires_grad=True), torch.ones(N, K, device='cuda'))


def test_infinities_in_the_gradient():
    """An infinity in dy: its row of dW is NaN where dy is split into parts (infinity less infinity), and in bf16 infinity times the
    values of x; other rows are as without it."""
    from spgt_b200 import ops
    for dtype in TYPES:
        x, dy = _rand(700, 64, seed=1, dtype=dtype), _rand(700, 40, seed=2, dtype=dtype)
        x[301, 5], x[301, 6], x[301, 7] = 0.0, 2.0, -2.0
        kept = ops.compress8(x)
        clean, clean_db = ops.weight_gradient8(dy, kept)
        dy[301, 9] = float('inf')
        dy[301, 11] = float('-inf')
        dw, db = ops.weight_gradient8(dy, kept)
        if dtype == torch.bfloat16:
            want = float('inf') * _kept64(x)[301]               # (zero times infinity is NaN)
            assert want[5].isnan() and want[6] == float('inf') and want[7] == float('-inf')
            for row, sign in ((9, 1), (11, -1)):
                assert torch.equal(dw[row].isnan(), want.isnan()) and torch.equal(dw[row].double().nan_to_num(0, 1, -1), (sign * want).nan_to_num(0, 1, -1))
        else:
            assert dw[9].isnan().all() and dw[11].isnan().all()
        rest = [i for i in range(40) if i not in (9, 11)]
        assert torch.equal(dw[rest], clean[rest]) and torch.equal(db[rest], clean_db[rest])
        assert db[9] == float('inf') and db[11] == float('-inf')


# ---------------------------------------------------------------------------------------------------------------------------------
# several units of samples
# ---------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype,C,G', [(torch.bfloat16, 128, 8), (torch.bfloat16, 130, 10), (torch.float16, 130, 26), (torch.float32, 130, 10)])
def test_group_norm_units_in_every_type(dtype, C, G):
    """At least three units of samples either way, among them samples that start off a 16-byte boundary and checkpoints whose blocks two
    samples share; forward out of place and in place."""
    from spgt_b200 import ops
    from spgt_b200._lib import lib
    N, P = 27, 181 * 181
    for tensors in (2, 3, 4):                                   # bytes that both passes read, in units of 96 MB
        assert -(-N // ((96 << 20) // (P * C * tensors))) >= 3
    x, dy = _rand(N, P, C, seed=1, mean=0.3, dtype=dtype), _rand(N, P, C, seed=2, dtype=dtype)
    w, b = _rand(C, seed=3, mean=1.0, scale=0.2), _rand(C, seed=4)
    y, stats, kept = ops.group_norm(x, G, w, b, 1e-5, 'silu', compress=True)
    dx, dw, db = ops.group_norm_backward(dy, x, G, w, b, stats, 'silu')
    dx8, dw8, db8 = ops.group_norm_backward(dy, kept, G, w, b, stats, 'silu')
    assert torch.equal(kept.codes, ops.compress8(x).codes) and torch.equal(kept.steps, ops.compress8(x).steps)
    x8 = _kept64(x)
    sums = [torch.zeros(2, C, device='cuda', dtype=torch.float64) for _ in range(4)]
    for n in range(N):
        want = _norm64(x[n:n + 1], G, w, b, 1e-5, 'silu', dy[n:n + 1])
        want8 = _norm64(x[n:n + 1], G, w, b, 1e-5, 'silu', dy[n:n + 1], x8[n:n + 1])
        for got, (value, tol) in ((y, want['y']), (dx, want['dx']), (dx8, want8['dx'])):
            _within(got[n:n + 1], value, tol + _rounded(value, dtype))
        for s, v in zip(sums, (want['dw'], want['db'], want8['dw'], want8['db'])):
            s += torch.stack(v)
    # a sample's tolerance has 100 roundings of the magnitudes' sum; a thread's chain of up to 90 values, the 12 to 16 sets of a tile, and
    # then chains of 27 * 148 / 128 tiles and 13 merges are below twice that
    for got, (value, tol) in zip((dw, db, dw8, db8), sums):
        _within(got, value, 2 * tol)
    need, code = lib.spgt_group_norm_workspace_bytes(N, P, C, G, ops.DTYPE[dtype]), ops.DTYPE[dtype]
    ws = torch.empty(need, dtype=torch.uint8, device='cuda')
    s = torch.empty_like(stats)
    rc = lib.spgt_group_norm_fwd(x.data_ptr(), w.data_ptr(), b.data_ptr(), x.data_ptr(), s.data_ptr(), None, None, N, P, C, G, 1e-5, 2, code,
                                 ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(x, y) and torch.equal(s, stats)


# ---------------------------------------------------------------------------------------------------------------------------------
# weight gradients of long blocks
# ---------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,N,K', [(179776, 256, 128), (179776, 256, 512), (400000, 8, 16), (400001, 16, 240), (400000, 5, 9), (400001, 9, 130)])
def test_weight_gradient8_many_chains(dtype, rows, N, K):
    """Blocks of 2400 to 4900 rows: two to four times 1280, after which an accumulator's sum moves to memory and it starts again."""
    from spgt_b200 import ops
    splits = max(1, torch.cuda.get_device_properties(0).multi_processor_count // (-(-N // 128) * (1 if K <= 128 else -(-K // 256))))
    assert rows / splits > 1280
    x, dy = _rand(rows, K, seed=1, dtype=dtype, mean=0.5), _rand(rows, N, seed=2, dtype=dtype)
    kept = ops.compress8(x)
    dw, db = ops.weight_gradient8(dy, kept)
    v, d = _kept64(x), dy.double()
    # 80 additions that truncate (2 U each) before a sum moves on, at most 4 such sums, and 148 / 16 blocks' results in a row, then 15
    _within(dw, d.t() @ v, 192 * U * (d.abs().t() @ v.abs()) + 1e-37)
    # a thread's chain of at most rows / (16 splits) values, 32 threads, and the blocks as above
    _within(db, d.sum(0), (rows / (16 * splits) + 64) * U * d.abs().sum(0))
    again = ops.weight_gradient8(dy, kept)
    assert torch.equal(again[0], dw) and torch.equal(again[1], db)


# ---------------------------------------------------------------------------------------------------------------------------------
# the convolution before a normalisation
# ---------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('bits', [32, 8])
def test_convolution_bias_before_a_normalisation(bits):
    """Sums of dx over a channel's pixels.  The norm takes out what a group's channels have in common, not these sums: their mean size is that of
    dozens of pixels.  1798 pixels of dx, each off by at most 100 U of its terms, which are below 4 in the mean, and summed in fp32: below 0.06 in
    the worst case; as independent roundings of 2 U each below 1e-4 of 30 in all, of which 1e-5 allows three times."""
    from spgt_b200.network.layer import ConvResBlock2D
    torch.manual_seed(0)
    block = ConvResBlock2D(6, 42, 3, 1, 0.0, 'silu', num_group=8).cuda()
    block.norm.activation_bits = bits
    x = _rand(2, 6, 31, 29, seed=5).requires_grad_()
    dy = _rand(2, 42, 31, 29, seed=6)
    with torch.backends.cudnn.flags(allow_tf32=False, deterministic=True):
        got, = torch.autograd.grad(block.forward_train(x), block.conv_layer.bias, dy)
        z = block.conv_layer(x).detach().permute(0, 2, 3, 1).contiguous()
    w, b = block.norm.weight.detach(), block.norm.bias.detach()
    want = _norm64(z, 7, w, b, 1e-5, 'silu', dy.permute(0, 2, 3, 1).contiguous(), _kept64(z) if bits == 8 else None)['dx'][0].sum((0, 1, 2))
    assert float(want.abs().mean()) > 10 and rel_l2(got, want) < 1e-5
