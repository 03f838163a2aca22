"""GroupNorm + activation, channels last: forward, backward and the form that ends in 8-bit blocks, against 64 bits.

Tolerances, from the arithmetic: per element xh is (x - mean) rstd, two float32 operations on a mean that is itself rounded to
float32, so |error(xh)| <= 2^-24 (2 |xh| + |mean| rstd) + the error of rstd (2^-23 |xh|): a few 2^-24 of 1 + |mean| rstd.  The
activation adds a few units in the last place; 1e-6 (1 + |mean| rstd) of the norm covers float32.  16-bit outputs: plus half a step
(finfo.eps / 2).  Gradients are sums of such terms: 4e-6 of the norm."""
import pytest
import torch
import torch.nn.functional as F

from helpers import rel_l2

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SLOPE = 0.1


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a ROCm GPU")
    from preset_gen_vae_amd import _lib, ops as _ops
    _lib.load()
    return _ops


def acts(ops):
    return {'none': (ops.PGV_ACT_NONE, lambda u: u), 'leaky': (ops.PGV_ACT_LEAKY_RELU, lambda u: F.leaky_relu(u, SLOPE)),
            'hardtanh': (ops.PGV_ACT_HARDTANH, lambda u: F.hardtanh(u)), 'silu': (ops.PGV_ACT_SILU, F.silu)}


def make(N, P, C, dtype, seed=0, mean=0.5, affine=True):
    g = torch.Generator().manual_seed(seed + 7919 * N + 31 * P + C)
    x = torch.randn(N, P, C, generator=g) * torch.exp(0.3 * torch.randn(C, generator=g)) + mean * torch.randn(N, 1, C, generator=g)
    gy = torch.randn(N, P, C, generator=g)
    w = 1 + 0.2 * torch.randn(C, generator=g) if affine else None
    b = 0.2 * torch.randn(C, generator=g) if affine else None
    return x.to(dtype), gy.to(dtype), w, b


def reference(x, gy, G, w, b, eps, act):
    """float64, torch's own group norm on the transposed tensor and autograd."""
    xr = x.double().requires_grad_(True)
    wr, br = (None if t is None else t.double().requires_grad_(True) for t in (w, b))
    y = act(F.group_norm(xr.transpose(1, 2), G, wr, br, eps)).transpose(1, 2)
    y.backward(gy.double())
    v = xr.detach().view(x.shape[0], x.shape[1], G, -1)
    mean = v.mean((1, 3))
    rstd = 1 / torch.sqrt(v.var((1, 3), unbiased=False) + eps)
    return y.detach(), mean, rstd, xr.grad, None if w is None else wr.grad, None if b is None else br.grad


def kinks_away(x, G, w, b, eps, act, margin):
    """Values whose pre-activation lies within `margin` of a kink are moved: which side they fall on is decided by rounding."""
    if act not in ('leaky', 'hardtanh'):
        return x
    for _ in range(4):
        u = F.group_norm(x.double().transpose(1, 2), G, None if w is None else w.double(), None if b is None else b.double(), eps)
        near = (u.transpose(1, 2).abs() - (0.0 if act == 'leaky' else 1.0)).abs() < margin
        if not near.any():
            break
        x = torch.where(near, (x.float() + 0.05).to(x.dtype), x).contiguous()
    return x


def check(ops, x, gy, G, w, b, act, eps=1e-5):
    code, f = acts(ops)[act]
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    y, mean, rstd = ops.group_norm_act_fwd(x.cuda(), G, dev(w), dev(b), eps, code, SLOPE)
    yr, mr, rr, gxr, gwr, gbr = reference(x, gy, G, w, b, eps, f)
    far = 1.0 + float((mr.abs() * rr).max())
    half = 0.0 if x.dtype == torch.float32 else torch.finfo(x.dtype).eps / 2
    assert y.dtype == x.dtype and rel_l2(y, yr) <= 1e-6 * far + half
    assert ((mean.double().cpu() - mr).abs() <= 1e-6 * (mr.abs() + 1 / rr)).all()
    assert ((rstd.double().cpu() / rr - 1).abs() <= 1e-6 * far).all()
    gx, gw, gb = ops.group_norm_act_bwd(gy.cuda(), x.cuda(), mean, rstd, G, dev(w), dev(b), code, SLOPE)
    assert gx.dtype == x.dtype
    if gxr.norm() > 1e-9 * gy.double().norm() * rr.max():      # (a group of one value has no gradient)
        assert rel_l2(gx, gxr) <= 4e-6 * far + half
    if w is not None:
        # sums of n terms: n 2^-24 of the sum of their magnitudes at most; 4e-6 of the norm in practice
        assert rel_l2(gw, gwr) <= 4e-6 * far and rel_l2(gb, gbr) <= 4e-6 * far
    again = ops.group_norm_act_bwd(gy.cuda(), x.cuda(), mean, rstd, G, dev(w), dev(b), code, SLOPE)
    assert torch.equal(again[0], gx) and torch.equal(again[1], gw) and torch.equal(again[2], gb)


# (items, pixels, channels, groups): groups of 8 k and of odd widths, rows that are not multiples of 16 bytes, one pixel, one
# group, every channel a group, slabs that fit a workgroup's registers and slabs that do not, more channels than a block has columns
SHAPES = [(1, 1, 32, 4), (1, 12, 2048, 32), (2, 391, 64, 8), (3, 17, 6, 3), (2, 33, 5, 1), (2, 40, 12, 12), (4, 1, 1024, 32),
          (2, 100, 24, 3), (1, 1485, 96, 4), (2, 5000, 32, 8), (1, 3000, 20, 5), (1, 9, 4104, 3), (1, 600, 2600, 2), (1, 70, 2304, 96),
          (2, 700, 256, 32), (1, 4100, 512, 32), (1, 2, 16400, 2),
          # one wave per workgroup (many small slabs), the largest slabs in registers, and slices of 128 partial sums
          (1100, 5, 32, 4), (300, 40, 128, 16), (2, 1485, 256, 16), (1, 1000, 64, 2), (2, 20000, 128, 4),
          # many items (parameter gradients in two levels), one or two pixels (several groups per wave)
          (2100, 1, 96, 3), (1030, 2, 20, 4), (70000, 1, 8, 2), (256, 1, 1024, 32)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_forward_and_backward(ops, shape, dtype):
    N, P, C, G = shape
    for act in ('silu', 'leaky') if P * C < 100000 else ('silu',):
        x, gy, w, b = make(N, P, C, dtype)
        check(ops, kinks_away(x, G, w, b, 1e-5, act, 1e-4), gy, G, w, b, act)


@pytest.mark.parametrize("act", ['none', 'leaky', 'hardtanh', 'silu'])
@pytest.mark.parametrize("shape", [(3, 50, 48, 6), (1, 2600, 64, 2)])
def test_activations_and_missing_affine(ops, shape, act):
    N, P, C, G = shape
    x, gy, w, b = make(N, P, C, torch.float32)
    code, f = acts(ops)[act]
    x = kinks_away(x, G, w, b, 1e-5, act, 1e-4)
    check(ops, x, gy, G, w, b, act)
    y, mean, rstd = ops.group_norm_act_fwd(x.cuda(), G, None, None, 1e-3, code, SLOPE)
    gxs = ops.group_norm_act_bwd(gy.cuda(), x.cuda(), mean, rstd, G, None, None, code, SLOPE, need_params=False)
    yr, _, _, gxr, _, _ = reference(x, gy, G, None, None, 1e-3, f)
    assert rel_l2(y, yr) <= 2e-6 and rel_l2(gxs[0], gxr) <= (8e-6 if act in ('none', 'silu') else 2e-2) and gxs[1] is None and gxs[2] is None


@pytest.mark.parametrize("shape", [(2, 391, 64, 8), (1, 6000, 64, 8), (2, 300, 24, 8)])
@pytest.mark.parametrize("mean", [30.0, 1000.0])
def test_large_means(ops, shape, mean):
    """Means far above the deviation: the variance must not come from a difference of 32-bit sums."""
    N, P, C, G = shape
    g = torch.Generator().manual_seed(5)
    x = torch.randn(N, P, C, generator=g) + mean
    x[:, 0] = 0.0             # an outlier where a shift might be taken from
    gy = torch.randn(N, P, C, generator=g)
    check(ops, x, gy, G, torch.ones(C), torch.zeros(C), 'silu')


def test_backward_against_differences(ops):
    """<gx, d>, <ggamma, d>, <gbeta, d> against central differences of the 64-bit forward pass (step 1e-4: truncation 1e-8,
    cancellation 1e-12), to the 4e-6 of the gradients' own arithmetic in the norm of the terms."""
    N, P, C, G = 2, 37, 24, 4
    x, gy, w, b = make(N, P, C, torch.float32)
    y, mean, rstd = ops.group_norm_act_fwd(x.cuda(), G, w.cuda(), b.cuda(), 1e-5, ops.PGV_ACT_SILU)
    grads = ops.group_norm_act_bwd(gy.cuda(), x.cuda(), mean, rstd, G, w.cuda(), b.cuda(), ops.PGV_ACT_SILU)

    def loss(x, w, b):
        return (F.silu(F.group_norm(x.transpose(1, 2), G, w, b, 1e-5)).transpose(1, 2) * gy.double()).sum()
    args = [t.double() for t in (x, w, b)]
    gen = torch.Generator().manual_seed(1)
    for k, grad in enumerate(grads):
        d = torch.randn(args[k].shape, generator=gen).double()
        up, down = [t.clone() for t in args], [t.clone() for t in args]
        up[k] += 1e-4 * d
        down[k] -= 1e-4 * d
        diff = (loss(*up) - loss(*down)) / 2e-4
        assert abs((grad.double().cpu() * d).sum() - diff) <= 1e-5 * grad.double().norm().cpu() * d.norm()


@pytest.mark.parametrize("shape", [(2, 40, 64, 8), (2, 5000, 64, 8), (1, 30, 12, 4)])
def test_non_finite_values_stay_in_their_group(ops, shape):
    N, P, C, G = shape
    x, gy, w, b = make(N, P, C, torch.float32)
    clean, mean, rstd = ops.group_norm_act_fwd(x.cuda(), G, w.cuda(), b.cuda())
    for bad in (float('nan'), float('inf')):
        x2 = x.clone()
        x2[0, P // 2, 0] = bad
        y, m2, r2 = ops.group_norm_act_fwd(x2.cuda(), G, w.cuda(), b.cuda())
        hit = torch.zeros(N, P, C, dtype=torch.bool, device='cuda')
        hit[0, :, :C // G] = True
        assert torch.isnan(y[hit]).all() and torch.equal(y[~hit], clean[~hit])
        gx, _, _ = ops.group_norm_act_bwd(gy.cuda(), x2.cuda(), m2, r2, G, w.cuda(), b.cuda())
        assert torch.isnan(gx[hit]).all() and torch.isfinite(gx[~hit]).all()


def test_constant_input(ops):
    """No variance: y = act(beta), and a gradient of 1 / sqrt(eps) steepness that stays finite."""
    x = torch.full((2, 50, 16), 3.25)
    y, mean, rstd = ops.group_norm_act_fwd(x.cuda(), 2, torch.ones(16).cuda(), torch.full((16,), 0.5).cuda(), 1e-5)
    assert (y == 0.5).all() and (mean == 3.25).all()
    gx, _, gb = ops.group_norm_act_bwd(torch.ones(2, 50, 16).cuda(), x.cuda(), mean, rstd, 2, torch.ones(16).cuda(), torch.zeros(16).cuda())
    assert gx.abs().max() < 1e-3 and torch.equal(gb, torch.full((16,), 100.0, device='cuda'))


def step_of(v, fmt):
    """Largest rounding error of an 8-bit code around the scaled value v."""
    man, emin = (3, -6) if fmt == 'e4m3' else (2, -14)
    e = torch.floor(torch.log2(v.abs().clamp_min(1e-30))).clamp_min(emin)
    return torch.exp2(e - man - 1)


@pytest.mark.parametrize("shape", [(1, 12, 2048, 32), (3, 20, 128, 8), (2, 33, 100, 4), (2, 50, 6, 3), (2, 3000, 256, 32), (1, 40, 2304, 12),
                                   (1, 700, 200, 5), (64, 1, 1024, 32), (1, 2200, 384, 4), (600, 9, 256, 8), (2, 1485, 256, 16),
                                   (1, 1400, 384, 12), (1, 1400, 130, 13)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_eight_bit_output(ops, shape, dtype):
    """Scales to float32 accuracy; every byte within half a step of the scaled 64-bit result (plus the 1e-6 of the value)."""
    N, P, C, G = shape
    x, _, w, b = make(N, P, C, dtype)
    for act, fmt in (('silu', 'e4m3'), ('leaky', 'e5m2')):
        code, f = acts(ops)[act]
        t = ops.group_norm_act_fp8(x.cuda(), G, w.cuda(), b.cuda(), 1e-5, code, SLOPE, fmt)
        y = f(F.group_norm(x.double().transpose(1, 2), G, w.double(), b.double(), 1e-5)).transpose(1, 2).reshape(N * P, C)
        kb = -(-C // 128)
        pad = F.pad(y, (0, kb * 128 - C)).view(N * P, kb, 128)
        s = pad.abs().amax(-1).clamp_min(2.0 ** -100) / (448.0 if fmt == 'e4m3' else 57344.0)
        got = t.scale.double().cpu().t()
        far = 4e-6 * 6
        assert t.cols == C and ((got / s - 1).abs() <= far).all()
        v = pad / s.unsqueeze(-1)
        q = t.q.double().cpu().view(N * P, kb, 128)
        assert ((q - v).abs() <= step_of(v * (1 + far), fmt) * (1 + far) + far * (v.abs() + v.abs().amax(-1, keepdim=True) * 0.02)).all()
        assert (q.flatten(1)[:, C:] == 0).all()


def test_block_of_the_three_operators(ops):
    """GroupNorm + activation -> 8-bit rows -> product, as a pointwise block runs, against its parts and against 64 bits."""
    from preset_gen_vae_amd.model import layer
    torch.manual_seed(3)
    norm, lin = layer.GroupNormAct(8, 256, activation=torch.nn.SiLU()).cuda(), layer.Fp8Linear(256, 136).cuda().eval()
    x = torch.randn(3, 256, 5, 7).cuda().to(memory_format=torch.channels_last)
    a = norm.forward_fp8(x)
    w = ops.fp8_quantize(lin.weight.detach(), 'tile')
    y = ops.fp8_matmul(a, w, lin.bias.detach(), torch.float32)
    ref = a.dequantize().double() @ w.dequantize().double().t() + lin.bias.double()
    assert y.shape == (105, 136) and rel_l2(y, ref) < 2e-6
    h = norm(x)
    assert h.shape == x.shape and h.is_contiguous(memory_format=torch.channels_last)
    z = lin(h.movedim(1, -1))
    # both round the same values to 8 bits; a value next to a tie may fall on either side (2^-4 of it, one in 10^4 values)
    assert rel_l2(z.reshape(105, 136), y) < 2.0 ** -4 * 1e-2 + 1e-6
    z.square().sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in [*norm.parameters(), *lin.parameters()])


def test_captured_training_step(ops):
    """Forward and backward of a small network of the modules in one graph, captured after a warm-up whose graphs are gone, replayed on
    new values with eager steps between: every gradient equals the eager one."""
    from preset_gen_vae_amd.model import layer
    torch.manual_seed(5)
    net = torch.nn.Sequential(layer.Fp8Linear(64, 128), layer.GroupNormAct(8, 128, activation=torch.nn.SiLU()),
                              layer.Fp8Linear(128, 32, grad_fmt='e5m2')).cuda()
    params = list(net.parameters())
    x, gy = torch.randn(40, 64, device='cuda'), torch.randn(40, 32, device='cuda')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            net.zero_grad(set_to_none=True)
            net(x).backward(gy)
    torch.cuda.current_stream().wait_stream(side)
    net.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = net(x)
        out.backward(gy)
    captured = [p.grad for p in params]
    out = out.detach()
    for rep in range(3):
        x.copy_(torch.randn(40, 64, generator=torch.Generator().manual_seed(rep)))
        gy.copy_(torch.randn(40, 32, generator=torch.Generator().manual_seed(rep + 9)))
        graph.replay()
        y = net(x)
        assert torch.equal(out, y)
        for a, b in zip(captured, torch.autograd.grad(y, params, gy)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("shape", [(2, 24, 9, 7), (3, 24), (2, 24, 11)])
def test_module(ops, shape):
    from preset_gen_vae_amd.model import layer
    torch.manual_seed(4)
    for act in (None, torch.nn.SiLU(), torch.nn.LeakyReLU(0.2), torch.nn.Hardtanh()):
        m = layer.GroupNormAct(4, 24, activation=act).cuda()
        torch.nn.init.normal_(m.weight)
        x = torch.randn(*shape).cuda().requires_grad_(True)
        y = m(x)
        y.square().sum().backward()
        ref = torch.nn.GroupNorm(4, 24).cuda().double()
        ref.load_state_dict(m.state_dict())
        xr = x.detach().double().requires_grad_(True)
        yr = ref(xr) if act is None else act(ref(xr))
        yr.square().sum().backward()
        assert rel_l2(y, yr) < 2e-6 and rel_l2(x.grad, xr.grad) < 1e-5
        assert rel_l2(m.weight.grad, ref.weight.grad) < 1e-5 and rel_l2(m.bias.grad, ref.bias.grad) < 1e-5
    with pytest.raises(ValueError, match="expected"):
        m(torch.randn(2, 25, 3).cuda())
    with pytest.raises(ValueError, match="divide"):
        layer.GroupNormAct(5, 24)
    with pytest.raises(NotImplementedError, match="epilogue"):
        layer.GroupNormAct(4, 24, activation=torch.nn.GELU())


def test_streams_graphs_and_neighbours(ops):
    """Another stream; captured graphs replayed in turn; the memory behind the outputs stays as it was."""
    sizes = [(2, 50, 64, 8), (1, 6000, 64, 8), (2, 31, 20, 4)]
    side = torch.cuda.Stream()
    graphs = []
    for N, P, C, G in sizes:
        x, gy, w, b = (t.cuda() for t in make(N, P, C, torch.bfloat16))

        def step(x=x, gy=gy, w=w, b=b, G=G):
            y, m, r = ops.group_norm_act_fwd(x, G, w, b, 1e-5, ops.PGV_ACT_SILU)
            t = ops.group_norm_act_fp8(x, G, w, b, 1e-5, ops.PGV_ACT_SILU)
            return (y, m, r, t.q.view(torch.uint8), t.scale) + ops.group_norm_act_bwd(gy, x, m, r, G, w, b, ops.PGV_ACT_SILU)
        eager = step()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(eager, other))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, x, gy, step, out))
    for rep in range(3):
        for graph, x, gy, step, out in graphs:
            xn, gn, _, _ = make(*x.shape, torch.bfloat16, seed=rep + 1)
            x.copy_(xn)
            gy.copy_(gn)
        for graph, *_ in graphs:
            graph.replay()
        for graph, x, gy, step, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, step()))


def test_empty_and_refused(ops):
    z = torch.zeros(0, 5, 8, device='cuda')
    y, m, r = ops.group_norm_act_fwd(z, 2)
    assert y.shape == (0, 5, 8) and m.shape == (0, 2)
    gx, gw, gb = ops.group_norm_act_bwd(z, z, m, r, 2)
    assert gx.shape == z.shape and (gw == 0).all() and (gb == 0).all()
    assert ops.group_norm_act_fp8(torch.zeros(3, 0, 8, device='cuda'), 2).q.shape == (0, 128)
    x = torch.randn(2, 5, 8, device='cuda')
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.group_norm_act_fwd(x.transpose(1, 2), 5)
    with pytest.raises(ValueError, match="divide"):
        ops.group_norm_act_fwd(x, 3)
    with pytest.raises(ValueError, match="activation"):
        ops.group_norm_act_fwd(x, 2, act=9)
    with pytest.raises(ValueError, match="weight"):
        ops.group_norm_act_fwd(x, 2, torch.ones(7, device='cuda'))
    with pytest.raises(RuntimeError, match="different devices"):
        ops.group_norm_act_fwd(x, 2, torch.ones(8))
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        ops.group_norm_act_fwd(x.double(), 2)
    _, m, r = ops.group_norm_act_fwd(x, 2)
    with pytest.raises(ValueError, match="like x"):
        ops.group_norm_act_bwd(x.bfloat16(), x, m, r, 2)
    with pytest.raises(ValueError, match="mean"):
        ops.group_norm_act_bwd(x, x, m[:1].contiguous(), r, 2)
