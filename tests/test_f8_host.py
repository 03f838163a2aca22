"""CPU: what the 8-bit and group-norm entry points refuse before any launch, and the modules built on them."""
import os

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from preset_gen_vae_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libpgv_hip.so not built")
    return _lib.load()


def refused(lib, rc, text, code=-1):
    assert rc == code and text in lib.pgv_last_error(), lib.pgv_last_error()


def test_quantize_arguments(lib):
    q = lambda x=16, dt=0, r=4, c=8, ld=8, block=0, fmt=0, p=16, s=16, pt=None, st=None, cs=None, ws=None, n=0: (  # noqa: E731
        lib.pgv_f8_quantize(x, dt, r, c, ld, block, fmt, p, s, pt, st, cs, ws, n, None))
    refused(lib, q(dt=3), b"element type")
    refused(lib, q(block=2), b"block kind")
    refused(lib, q(fmt=2), b"format")
    refused(lib, q(r=-1), b"extents")
    refused(lib, q(ld=7), b"row stride")
    refused(lib, q(s=None), b"come together")
    refused(lib, q(p=None, s=None), b"nothing to write")
    refused(lib, q(p=24), b"aligned")
    refused(lib, q(x=None), b"null input")
    refused(lib, q(r=1 << 24, c=1 << 20, ld=1 << 20), b"too large")
    refused(lib, q(cs=16), b"workspace", -3)
    refused(lib, q(cs=16, ws=16, n=31), b"workspace", -3)
    assert q(r=0) == 0 and q(c=0, ld=0) == 0
    assert lib.pgv_f8_quantize_workspace(129, 10) == 80 and lib.pgv_f8_quantize_workspace(0, 10) == 0


def test_product_arguments(lib):
    m = lambda M=4, N=4, K=8, a=16, sa=16, fa=0, b=16, sb=16, kind=1, out=16, dt=0, ws=None, n=0: (  # noqa: E731
        lib.pgv_f8_matmul(M, N, K, a, sa, fa, b, sb, kind, None, out, dt, ws, n, None))
    refused(lib, m(M=-1), b"extents")
    refused(lib, m(K=(1 << 23) + 1), b"extents")
    refused(lib, m(fa=2), b"format")
    refused(lib, m(kind=2), b"block kind")
    refused(lib, m(dt=5), b"output type")
    refused(lib, m(a=None), b"null operand")
    refused(lib, m(K=0), b"empty reduction")
    refused(lib, m(b=8), b"aligned")
    refused(lib, m(out=20), b"aligned")
    assert m(M=0) == 0 and m(N=0) == 0
    need = lib.pgv_f8_matmul_workspace(4, 64, 1 << 16, 1)
    assert need > 0
    refused(lib, m(N=64, K=1 << 16), b"workspace", -3)
    refused(lib, m(N=64, K=1 << 16, ws=16, n=need - 1), b"workspace", -3)
    assert lib.pgv_f8_linear(16, 0, 100, 8, 8, 16, 16, 1, 4, None, None, None, 16, 0, None, 0, None) == -1
    assert b"quantised rows" in lib.pgv_last_error()
    refused(lib, lib.pgv_f8_linear(16, 0, 1, 8, 7, 16, 16, 1, 4, None, None, None, 16, 0, None, 0, None), b"row stride")
    # a split reduction's workspace never exceeds its outputs times the splits, and grows with neither sign of the sizes
    for M, N, K in [(1, 1, 1), (1, 4096, 4096), (37, 1024, 24576), (256, 1024, 25024), (16384, 8192, 8192)]:
        for kind in (0, 1):
            assert lib.pgv_f8_matmul_workspace(M, N, K, kind) % (4 * M * N) == 0


def test_group_norm_arguments(lib):
    f = lambda x=16, dt=0, N=2, P=4, C=8, G=2, act=0, y=16, m=16, r=16, ws=None, n=0: (  # noqa: E731
        lib.pgv_group_norm_act_fwd(x, dt, N, P, C, G, None, None, 1e-5, act, 0.0, y, m, r, ws, n, None))
    refused(lib, f(dt=7), b"element type")
    refused(lib, f(act=4), b"activation")
    refused(lib, f(G=3), b"sizes")
    refused(lib, f(G=0), b"sizes")
    refused(lib, f(N=(1 << 24) + 1), b"too large")
    refused(lib, f(x=None), b"null")
    refused(lib, f(m=None), b"null")
    refused(lib, f(P=1 << 20), b"workspace", -3)
    assert f(N=0) == 0 and f(P=0) == 0
    refused(lib, lib.pgv_group_norm_act_f8(16, 0, 2, 4, 8, 2, None, None, 1e-5, 0, 0.0, 3, 16, 16, None, 0, None), b"8-bit format")
    refused(lib, lib.pgv_group_norm_act_f8(16, 0, 2, 4, 8, 2, None, None, 1e-5, 0, 0.0, 0, None, 16, None, 0, None), b"null")
    b = lambda ws=None, n=0, P=4, gg=16: lib.pgv_group_norm_act_bwd(16, 16, 0, 2, P, 8, 2, None, None, 16, 16, 0, 0.0, 16, gg, 16, ws, n, None)  # noqa: E731
    refused(lib, b(), b"workspace", -3)
    refused(lib, b(P=0), b"empty")
    assert lib.pgv_group_norm_workspace(2, 4, 8, 3, 0, 0) == 0 and lib.pgv_group_norm_workspace(2, 4, 8, 2, 0, 3) == 0


def test_no_cpu_path():
    from preset_gen_vae_amd import ops
    x = torch.ones(4, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.fp8_quantize(x)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.group_norm_act_fwd(x.view(1, 4, 8), 2)
    blocks = ops.Fp8Blocks(torch.zeros(4, 128, dtype=torch.float8_e4m3fn), torch.ones(1, 4), 'row', 8)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.fp8_matmul(blocks, blocks)
    # the values it stands for need no GPU
    assert torch.equal(blocks.dequantize(), torch.zeros(4, 8))


def test_modules_and_architecture_suffixes():
    from preset_gen_vae_amd.model import layer
    from preset_gen_vae_amd.model.regression import MLPRegression

    class Helper:
        learnable_preset_size = 21
    names = {a: list(MLPRegression(a, 16, Helper()).state_dict()) for a in ('2l64', '2l64_fp8', '2l64_gn', '2l64_gn_fp8')}
    assert names['2l64'] == names['2l64_fp8'] and names['2l64_gn'] == names['2l64_gn_fp8']
    assert [n.replace('gn1', 'bn1') for n in names['2l64_gn']] == [n for n in names['2l64'] if 'running' not in n and 'tracked' not in n]
    for bad in ('2l64_fp9', '2l64_fp8_fp8', '2l64_gn_x'):
        with pytest.raises(NotImplementedError, match="suffix"):
            MLPRegression(bad, 16, Helper())
    with pytest.raises(ValueError, match="grad_fmt"):
        layer.Fp8Linear(4, 4, grad_fmt='e3m4')
    assert layer.GroupNormAct(2, 8, affine=False).weight is None
