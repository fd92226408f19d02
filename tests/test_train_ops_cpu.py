"""What the entry points of group normalisation and 8-bit checkpoints refuse before anything is launched (no GPU needed: addresses
are checked, never read)."""
import pytest
import torch

OK, NULL, SHAPE, ALIGN, WORKSPACE = 0, -1, -2, -3, -4


def test_checkpoint_arguments():
    from spgt_b200._lib import lib
    for f in (lambda dtype=0, act=0, x=16, codes=32, steps=48, n=64: lib.spgt_compress8(x, dtype, act, None, codes, steps, n, None),
              lambda dtype=0, act=0, x=16, codes=32, steps=48, n=64: lib.spgt_restore8(codes, steps, None, act, x, dtype, n, None)):
        assert f(dtype=3) == f(dtype=-1) == f(act=4) == f(act=-1) == f(n=-1) == f(n=(1 << 38) + 1) == SHAPE
        assert f(x=None) == f(codes=None) == f(steps=None) == NULL
        assert f(x=24) == f(codes=40) == ALIGN
        assert f(n=0, x=None, codes=None, steps=None) == OK
    assert lib.spgt_compress8(16, 0, 1, 24, 32, 48, 64, None) == ALIGN
    assert lib.spgt_restore8(16, 32, 8, 1, 48, 0, 64, None) == ALIGN


def test_weight_gradient_arguments():
    from spgt_b200._lib import lib
    need = lib.spgt_weight_gradient8_workspace_bytes(128, 256, 4096)
    assert need > 0
    assert lib.spgt_weight_gradient8_workspace_bytes(0, 256, 4096) == lib.spgt_weight_gradient8_workspace_bytes(128, 0, 4096) == 0
    assert lib.spgt_weight_gradient8_workspace_bytes(128, 256, -1) == lib.spgt_weight_gradient8_workspace_bytes(16385, 1, 1) == 0
    f = lambda dy=16, dtype=0, codes=32, steps=48, dw=64, N=128, K=256, rows=4096, ws=128, size=need: lib.spgt_weight_gradient8(
        dy, dtype, codes, steps, dw, None, N, K, rows, ws, size, None)
    assert f(dtype=3) == f(N=0) == f(K=-1) == f(rows=-5) == SHAPE
    assert f(dy=None) == f(codes=None) == f(steps=None) == f(dw=None) == f(ws=None) == NULL
    assert f(size=need - 1) == WORKSPACE and f(dy=8) == f(codes=33) == f(ws=24) == ALIGN


def test_group_norm_arguments():
    from spgt_b200._lib import lib
    size, size_bwd = lib.spgt_group_norm_workspace_bytes, lib.spgt_group_norm_bwd_workspace_bytes
    for s in (size, size_bwd):
        assert s(4, 1849, 128, 8, 0) > 0 and s(4, 1849, 42, 7, 1) > 0 and s(1, 1, 2048, 1, 0) > 0 and s(1, 1, 4096, 1, 2) > 0 and s(1, 1, 511, 7, 1) > 0
        assert s(4, 1849, 128, 5, 0) == s(4, 1849, 0, 1, 0) == s(4, 1849, 128, 0, 0) == s(-1, 1849, 128, 8, 0) == s(4, -1, 128, 8, 0) == s(4, 1849, 128, 8, 3) == 0
        assert s(1, 1, 2052, 1, 0) == s(1, 1, 4104, 1, 1) == s(1, 1, 513, 1, 0) == 0 and s(1, 1 << 41, 1, 1, 0) == 0
    need = size(4, 1849, 128, 8, 0)
    f = lambda x=16, y=32, stats=48, codes=None, steps=None, C=128, G=8, act=2, dtype=0, ws=64, n=need: lib.spgt_group_norm_fwd(
        x, None, None, y, stats, codes, steps, 4, 1849, C, G, 1e-5, act, dtype, ws, n, None)
    assert f(G=3) == f(act=9) == f(dtype=7) == f(C=1001, G=1) == SHAPE
    assert f(x=None) == f(y=None) == f(stats=None) == f(ws=None) == f(codes=16) == f(steps=16) == NULL
    assert f(n=need - 1) == WORKSPACE and f(x=20) == f(y=40) == f(stats=8) == f(ws=72) == f(codes=8, steps=3) == ALIGN
    need = size_bwd(4, 1849, 128, 8, 0)
    f = lambda dy=16, x=32, codes=None, steps=None, stats=48, dx=64, G=8, act=2, dtype=0, ws=80, n=need: lib.spgt_group_norm_bwd(
        dy, x, codes, steps, None, None, stats, dx, None, None, 4, 1849, 128, G, act, dtype, ws, n, None)
    assert f(G=3) == f(act=9) == f(dtype=7) == SHAPE
    assert f(dy=None) == f(x=None) == f(stats=None) == f(dx=None) == f(ws=None) == f(codes=16) == NULL
    assert f(n=need - 1) == WORKSPACE and f(dy=20) == f(x=40) == f(dx=72) == f(stats=8) == f(ws=88) == f(codes=8, steps=3) == ALIGN


def test_no_cpu_path():
    from spgt_b200 import ops
    from spgt_b200.extension.bind.checkpoint8 import activation8
    from spgt_b200.extension.bind.normalization import group_norm_act
    x = torch.ones(2, 3, 8)
    for call in (lambda: group_norm_act(x, 2), lambda: activation8(x, 'relu'), lambda: ops.compress8(x),
                 lambda: ops.Checkpoint8(torch.zeros(48, dtype=torch.int8), torch.zeros(2, dtype=torch.uint8), x.shape)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError):
        group_norm_act(x, 2, activation_bits=16)
    with pytest.raises(TypeError):
        ops.compress8([1.0])
