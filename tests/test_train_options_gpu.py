"""The model with group normalisation in its scalers and with 8-bit activation checkpoints, in inference and in training."""
import numpy as np
import pytest
import torch

from tests.helpers import rel_l2

pytestmark = pytest.mark.gpu


def _config(**more):
    from spgt_b200.config.config_accessor import get_darcy_config
    from spgt_b200.dataset.darcy_dataset import GaussNormalizer
    cfg = get_darcy_config(3, 6, num_frequence_mode=4, clamp_attn=False, fine_resolution=85, num_encoder_layer=2, **more)
    cfg['target_normalizer'] = GaussNormalizer()
    return cfg


def _model(seed=3, **more):
    from spgt_b200.network.sp_model import Sp_GalerkinTransformer2D
    torch.manual_seed(seed)
    model = Sp_GalerkinTransformer2D(_config(**more)).cuda()
    with torch.no_grad():
        for name, p in model.named_parameters():
            if 'norm_layer' in name:
                p.add_(0.2 * torch.randn_like(p))
    return model


def _inputs(n=2, seed=0):
    from spgt_b200.dataset.darcy_dataset import meshgrid
    g = torch.Generator().manual_seed(seed)
    node = torch.where(torch.randn(n, 29, 29, 1, generator=g) > 0, 12.0, 3.0)
    grid = torch.rand(n, 29, 29, 2, generator=g)
    position = torch.rand(n, 15, 15, 2, generator=g)
    return node.cuda(), position.cuda(), grid.cuda()


def test_model_without_the_options_is_unchanged():
    model = _model()
    assert not any('norm_layer' in k for k in model.state_dict())
    node, position, grid = _inputs()
    model.eval()
    a = model(node, position, grid)
    assert model._plan is not None                             # the one-call forward
    assert _model(num_norm_group=8).down_scaler.conv1.norm.num_groups == 7       # (42 channels)


@pytest.mark.parametrize('act', ['relu', 'silu'])
def test_normalised_scalers_inference_follows_training(act):
    model = _model(num_norm_group=8, acti_downscaler=act)
    node, position, grid = _inputs()
    with torch.backends.cudnn.flags(allow_tf32=False):
        model.train()
        want = model(node, position, grid).detach()
        model.eval()
        got = model(node, position, grid)
    assert rel_l2(got, want) < 1e-4                            # the two paths' bound without the option, too
    assert rel_l2(got, _model(acti_downscaler=act).eval()(node, position, grid)) > 1e-3
    with torch.no_grad():                                      # new parameters are seen
        model.up_scaler.conv.norm.bias.add_(1.0)
    assert rel_l2(model(node, position, grid), got) > 1e-6


def test_normalised_block_gradients():
    """ConvResBlock2D with a normalisation against torch autograd in 64 bits.  1e-5: the library's fp32 convolution and its gradients."""
    from spgt_b200.network.layer import ConvResBlock2D
    torch.manual_seed(0)
    block = ConvResBlock2D(6, 42, 3, 1, 0.0, 'silu', num_group=8).cuda()
    x = torch.randn(2, 6, 31, 29, device='cuda', requires_grad=True)
    dy = torch.randn(2, 42, 31, 29, device='cuda')
    with torch.backends.cudnn.flags(allow_tf32=False):
        y = block.forward_train(x)
        got = [y, *torch.autograd.grad(y, [x, *block.parameters()], dy)]
    ref = [t.detach().double().requires_grad_() for t in (x, *block.parameters())]
    names = [n for n, _ in block.named_parameters()]
    p = dict(zip(names, ref[1:]))
    z = torch.nn.functional.conv2d(ref[0], p['conv_layer.weight'], p['conv_layer.bias'], padding=1)
    z = torch.nn.functional.silu(torch.nn.functional.group_norm(z, 7, p['norm_layer.weight'], p['norm_layer.bias'], 1e-5))
    want = [z, *torch.autograd.grad(z, ref, dy.double())]
    for name, a, b in zip(['y', 'x', *names], got, want):
        if name == 'conv_layer.bias':                          # (the norm takes out a group's common part: sums that nearly cancel)
            assert float((a.double() - b).abs().max()) < 1e-5 * float(dy.abs().sum())
        else:
            assert rel_l2(a, b) < 1e-5, name


def _step(model, inputs):
    model.train()
    model.zero_grad(set_to_none=True)
    out = model(*inputs)
    out.square().mean().backward()
    return out.detach(), {n: p.grad.clone() for n, p in model.named_parameters()}


def test_checkpoints_keep_values_and_nearly_gradients():
    """The forward pass with 8-bit checkpoints is the forward pass; every rounding to 8 bits is off by 1/127 of a block's largest value
    at most, and a gradient feels a few of them in a row: below a tenth of it, where a wrong one would be off by its own size."""
    inputs = _inputs()
    plain, kept = _model(num_norm_group=8, acti_encoder_ffn='silu'), _model(num_norm_group=8, acti_encoder_ffn='silu', activation_bits=8)
    kept.load_state_dict(plain.state_dict())
    assert kept.down_scaler.conv2.norm.activation_bits == 8 and kept.encoder_mixer.layers[0].ffn_layer.activation_bits == 8
    with torch.backends.cudnn.flags(allow_tf32=False):
        (a, ga), (b, gb) = _step(plain, inputs), _step(kept, inputs)
    assert rel_l2(b, a) < 1e-5
    for name in ga:
        if not name.endswith('conv_layer.bias'):
            assert rel_l2(gb[name], ga[name]) < 0.1, name
    assert any(not torch.equal(ga[n], gb[n]) for n in ga)


def test_feed_forward_memory_and_hooks():
    from spgt_b200.network.layer import FeedForward
    ffn = FeedForward(128, 128, 256, 0.0, 'silu').cuda()
    x = torch.randn(16, 4096, 128, device='cuda', requires_grad=True)

    def held(bits):
        ffn.activation_bits = bits
        before = torch.cuda.memory_allocated()
        y = ffn.forward_train(x)
        size = torch.cuda.memory_allocated() - before - y.numel() * 4
        g = torch.autograd.grad(y.square().sum(), (x, *ffn.parameters()))
        return size, y.detach(), g
    (full, a, ga), (small, b, gb) = held(32), held(8)
    rows = 16 * 4096
    assert full >= rows * 512 * 4 and small <= rows * 640 * 1.04     # hidden values before and after the activation; all three inputs in 8 bits
    assert rel_l2(b, a) < 1e-5                                 # (SiLU from the hardware exponential, 1e-6, against the library's)
    for u, v in zip(ga, gb):
        assert rel_l2(v, u) < 0.05
    seen = []
    handle = ffn.layer1.register_forward_hook(lambda *a: seen.append(1))
    ffn.forward_train(x)
    handle.remove()
    assert seen                                                # a hook sees the layer's call as without the option


def test_mixed_precision_step():
    model = _model(num_norm_group=8, activation_bits=8, acti_encoder_ffn='silu')
    ffn, norm = model.encoder_mixer.layers[0].ffn_layer, model.up_scaler.conv.norm
    x = torch.randn(2, 225, 128, device='cuda', requires_grad=True)
    with torch.autocast('cuda', dtype=torch.bfloat16):
        y = norm(ffn.forward_train(x))
        assert y.dtype == torch.bfloat16
    y.float().square().sum().backward()
    assert x.grad.dtype == torch.float32 and x.grad.isfinite().all()
    for p in (*ffn.parameters(), *norm.parameters()):
        assert p.grad.dtype == torch.float32 and p.grad.isfinite().all()


def test_training_run_with_the_options():
    """darcy_train with both options: it runs, and the saved state loads."""
    from spgt_b200.config.config_accessor import get_darcy_config
    from spgt_b200.network.sp_model import Sp_GalerkinTransformer2D
    from spgt_b200.run.darcy_train import darcy_train
    rng = np.random.default_rng(5)
    a = np.where(rng.standard_normal((4, 85, 85)) >= 0, 12.0, 3.0).astype(np.float32)
    data = {'a': a, 'u': (0.01 * rng.standard_normal((4, 85, 85))).astype(np.float32)}
    cfg = get_darcy_config(3, 6, num_frequence_mode=4, clamp_attn=False, fine_resolution=85, num_encoder_layer=2, num_data=4, batch_size=2, epochs=2,
                           seed=7, num_norm_group=4, activation_bits=8)
    ckpt = darcy_train(cfg, data, data, num_valid=2, log=None)
    assert np.isfinite(ckpt['loss_history']).all() and len(ckpt['loss_history']) == 2
    Sp_GalerkinTransformer2D(_config(num_norm_group=4)).load_state_dict(ckpt['Module'])


def test_bad_options():
    with pytest.raises(ValueError):
        _model(activation_bits=4)
