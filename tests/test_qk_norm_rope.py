"""Query/key norm with the position rotation: against the formula in 64
bits, both layouts, every stride, its gradients and refusals."""
import pytest
import torch

from pytorch_distributed_train_amd.ops import functional as OF

gpu = pytest.mark.gpu
DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=gpu)]
U = 2.0 ** -24


def _oracle(x, w, cos, sin, pos, eps, inter, dy=None):
    """64-bit y, and with dy the gradients, by complex numbers."""
    x = x.detach().double().cpu().requires_grad_(dy is not None)
    y, w64 = x, None
    if w is not None:
        w64 = w.detach().double().cpu().requires_grad_(dy is not None)
        y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w64
    if cos is not None:
        e = torch.complex(cos.double().cpu(), sin.double().cpu())
        s, half = x.shape[1], cos.shape[1]
        at = torch.arange(s).expand(x.shape[0], s) if pos is None \
            else pos.long().cpu()
        e = e[at][:, :, None]
        r = y[..., :2 * half]
        if inter:
            z = torch.view_as_complex(r.unflatten(-1, (half, 2))
                                      .contiguous()) * e
            r = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(r[..., :half], r[..., half:]) * e
            r = torch.cat([z.real, z.imag], -1)
        y = torch.cat([r, y[..., 2 * half:]], -1)
    if dy is None:
        return y, None, None
    g = torch.autograd.grad(y, (x,) if w is None else (x, w64),
                            dy.double().cpu())
    return y.detach(), g[0], g[1] if w is not None else None


def _check(got, want, dtype, size, what):
    """One rounding to the type (half a step, relative) beside fp32 work:
    under 40 roundings on values of at most `size` (a turned pair's terms
    may cancel, so they count by their size and not by the result's)."""
    half = torch.finfo(dtype).eps / 2
    bound = want.abs() * half * (1 + 2.0 ** -10) + 40 * U * size
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25  # half of the least step
    off = (got.detach().double().cpu() - want).abs()
    assert bool((off <= bound).all()), \
        f"{what}: {float((off - bound).max())} over the bound"


def _case(dev, dtype, b, s, h, hk, hd, rot, inter, pos, norm, pad=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    width = h + 2 * hk
    base = torch.randn(b, s, width, hd + pad, generator=g)
    base = (base * 1.5).to(dtype).to(dev)[..., :hd]
    q, k = base[:, :, :h], base[:, :, h:h + hk]
    wq = wk = cos = sin = p = None
    if norm:
        wq, wk = (1 + 0.2 * torch.randn(2, hd, generator=g)).to(dev)
    if rot:
        n = max(s, 300)
        cos, sin = OF.rope_tables(n, rot, device=dev)
        if pos:
            p = torch.randint(0, n, (b, s), generator=g).to(dev, pos)
    dq = torch.randn(b, s, h, hd, generator=g).to(dtype).to(dev)
    dk = torch.randn(b, s, hk, hd, generator=g).to(dtype).to(dev)
    return q, k, wq, wk, cos, sin, p, dq, dk


CASES = [
    # b, s, h, hk, hd, rot, inter, positions, norm, pad
    (2, 197, 12, 12, 64, 64, False, None, True, 0),
    (1, 1, 16, 4, 128, 128, False, torch.int64, True, 0),
    (3, 50, 6, 2, 128, 64, True, torch.int32, True, 0),
    (2, 33, 5, 1, 80, 32, False, None, True, 0),
    (2, 33, 3, 3, 96, 96, True, None, False, 0),   # rotation alone
    (2, 40, 4, 2, 64, 0, False, None, True, 0),    # norm alone
    (1, 130, 8, 8, 32, 32, False, None, True, 0),
    (1, 9, 2, 1, 256, 256, False, None, True, 0),
    (1, 9, 2, 1, 248, 128, True, None, True, 0),
    (2, 17, 3, 1, 8, 8, True, None, True, 0),
    # what 8-element lanes cannot load
    (2, 21, 3, 2, 64, 64, False, None, True, 3),   # rows off by 3 elements
    (2, 21, 3, 2, 72, 24, False, None, True, 0),   # halves of 12
    (2, 21, 3, 2, 50, 14, True, torch.int64, True, 0),
    (1, 5, 2, 2, 255, 254, False, None, True, 1),
    (1, 7, 2, 1, 1, 0, False, None, True, 0),
    (1, 4099, 2, 1, 64, 64, False, None, True, 0),
]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16,
                                   torch.float32])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_backward(dev, dtype, case):
    b, s, h, hk, hd, rot, inter, pos, norm, pad = case
    q, k, wq, wk, cos, sin, p, dq, dk = _case(
        dev, dtype, b, s, h, hk, hd, rot, inter, pos, norm, pad, seed=s + hd)
    leaves = [x.detach().requires_grad_(True) if x is not None else None
              for x in (q, k, wq, wk)]
    yq, yk = OF.qk_norm_rope(*leaves, cos, sin, positions=p,
                             interleaved=inter)
    assert yq.is_contiguous() and yq.dtype == dtype and yk.shape == k.shape
    live = [x for x in leaves if x is not None]
    grads = dict(zip([i for i, x in enumerate(leaves) if x is not None],
                     torch.autograd.grad((yq, yk), live, (dq, dk))))
    for i, (x, w, y, dy) in enumerate(((q, wq, yq, dq), (k, wk, yk, dk))):
        wy, wx, ww = _oracle(x, w, cos, sin, p, 1e-6, inter, dy)
        x64 = x.double().cpu()
        r = (x64.square().mean(-1, keepdim=True) + 1e-6).rsqrt() \
            if norm else torch.ones_like(x64[..., :1])
        top = 1.0 if w is None else float(w.abs().max())
        # a pair's larger element bounds both terms of a turn
        size = (x64 * r).abs().amax(-1, keepdim=True) * top * 2
        _check(y, wy, dtype, size, "y")
        g = dy.double().cpu().abs().amax(-1, keepdim=True) * top * 2
        xh = (x64 * r).abs()
        mean = (xh * g).mean(-1, keepdim=True)
        _check(grads[i], wx, dtype, r * (g + xh * mean), "dx")
        if w is not None:
            # a sum of b*s*heads products g * xhat: each off by 40
            # roundings, and sums of n of them by (log2 n + chain) more
            n = (xh * g).sum((0, 1, 2))
            off = (grads[i + 2].double().cpu() - ww).abs()
            assert bool((off <= n * U * (40 + 256)).all()), "dw"


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_gradients_against_differences(inter, norm):
    g = torch.Generator().manual_seed(4)
    q = torch.randn(2, 3, 2, 6, generator=g, dtype=torch.float64)
    k = torch.randn(2, 3, 1, 6, generator=g, dtype=torch.float64)
    w = [torch.rand(6, generator=g, dtype=torch.float64) + 0.5
         for _ in range(2)] if norm else [None, None]
    cos, sin = OF.rope_tables(5, 4)
    pos = torch.tensor([[0, 4, 2], [1, 1, 3]])
    leaves = [x.requires_grad_(True) for x in (q, k, *w) if x is not None]

    def f(*a):
        a = list(a) + [None] * (4 - len(a))
        return OF.qk_norm_rope(*a, cos.double(), sin.double(), positions=pos,
                               interleaved=inter)

    assert torch.autograd.gradcheck(f, leaves, eps=1e-6, atol=1e-6)


def test_tables():
    cos, sin = OF.rope_tables(100001, 64, theta=5e5, scale=2.0)
    i = 13
    a = 100000 / 2.0 * 5e5 ** (-2 * i / 64)
    assert abs(float(cos[100000, i]) - torch.tensor(
        a, dtype=torch.float64).cos()) <= 2 * U
    assert cos.shape == (100001, 32) and cos.dtype == torch.float32
    with pytest.raises(ValueError):
        OF.rope_tables(4, 3)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("hd", [64, 50])  # 8-element lanes, and the others
def test_position_outside_the_tables_shows(dev, hd):
    q = torch.ones(1, 4, 2, hd, device=dev)
    cos, sin = OF.rope_tables(3, 16, device=dev)
    pos = torch.tensor([[0, 3, -1, 2]], device=dev)
    y, _ = OF.qk_norm_rope(q, q, None, None, cos, sin, positions=pos)
    bad = torch.isnan(y[..., :16]).all(-1).all(-1).cpu()[0]
    assert bad.tolist() == [False, True, True, False]
    assert bool((y[..., 16:] == 1).all())


@pytest.mark.parametrize("dev", DEVICES)
def test_broadcast_inputs_and_gradients(dev):
    """Expanded inputs and the expanded gradient of a sum: zero strides."""
    x = torch.randn(1, 1, 1, 64, device=dev).requires_grad_(True)
    w = torch.ones(64, device=dev)
    cos, sin = OF.rope_tables(8, 64, device=dev)
    q = x.expand(2, 8, 3, 64)
    yq, yk = OF.qk_norm_rope(q, q, w, w, cos, sin)
    (yq.sum() + 2 * yk.sum()).backward()
    x64 = x.detach().double().cpu().requires_grad_(True)
    c, s = cos.double().cpu()[None, :, None], sin.double().cpu()[None, :, None]
    n = x64.expand(2, 8, 3, 64)
    n = n / (n.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    y = torch.cat([n[..., :32] * c - n[..., 32:] * s,
                   n[..., 32:] * c + n[..., :32] * s], -1)
    (3 * y.sum()).backward()
    # 96 heads' gradients, each off by 40 roundings of at most 4 * max|x|^2
    r = float(1 / x.detach().square().mean().sqrt())
    top = float(x.detach().abs().max()) ** 2 * r * r + 1
    bound = 2 * 96 * 40 * U * 4 * r * top
    assert float((x.grad.double().cpu() - x64.grad).abs().max()) <= bound


@pytest.mark.parametrize("dev", DEVICES)
def test_empty(dev):
    w = torch.ones(64, device=dev).requires_grad_(True)
    q = torch.zeros(0, 5, 2, 64, device=dev).requires_grad_(True)
    yq, yk = OF.qk_norm_rope(q, q, w, w)
    (yq.sum() + yk.sum()).backward()
    assert yq.shape == q.shape and float(w.grad.abs().max()) == 0.0
    k = torch.zeros(1, 5, 0, 64, device=dev)
    y, z = OF.qk_norm_rope(torch.ones(1, 5, 2, 64, device=dev), k, w.detach(),
                           w.detach())
    assert z.numel() == 0 and bool(torch.isfinite(y).all())


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    def z(*s, dt=torch.float32):
        return torch.zeros(*s, device=dev, dtype=dt)

    q, k, w = z(2, 4, 3, 64), z(2, 4, 1, 64), z(64)
    cos = z(4, 32)
    for a, kw in (
            ((q, z(2, 5, 1, 64), w, w), {}),
            ((q, z(2, 4, 1, 32), w, w), {}),
            ((q[0], k[0], w, w), {}),
            ((q, k.half(), w, w), {}),
            ((q, k), {}),
            ((q, k, w), {}),
            ((q, k, z(32), w), {}),
            ((q, k, w, w, cos), {}),
            ((q, k, w, w, cos, z(4, 16)), {}),
            ((q, k, w, w, z(4, 33), z(4, 33)), {}),
            ((q, k, w, w, z(3, 32), z(3, 32)), {}),
            ((q, k, w, w, cos, cos), {"positions": z(2, 4)}),
            ((q, k, w, w, cos, cos),
             {"positions": z(1, 4, dt=torch.int64)}),
            ((q, k, w, w, cos.clone().requires_grad_(True), cos), {}),
            ((z(1, 1, 1, 257), z(1, 1, 1, 257), z(257), z(257)), {})):
        with pytest.raises((ValueError, RuntimeError)):
            OF.qk_norm_rope(*a, **kw)


@gpu
def test_refuses_what_the_kernel_cannot_take():
    q = torch.zeros(2, 4, 3, 64, device="cuda")
    w = torch.zeros(64, device="cuda")
    for a in ((q.double(), q.double(), w, w),
              (q, q, w.half(), w.half()),
              (q, q, w.cpu(), w.cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            OF.qk_norm_rope(*a)


@gpu
def test_captured_and_on_another_stream():
    """Forward and backward replayed with new inputs, eager work between."""
    q, k, wq, wk, cos, sin, _, dq, dk = _case(
        "cuda", torch.bfloat16, 2, 65, 6, 2, 64, 64, False, None, True)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, wq, wk)]

    def step():
        y = OF.qk_norm_rope(*leaves, cos, sin)
        grads = torch.autograd.grad(y, leaves, (dq, dk))
        return [x.detach() for x in (*y, *grads)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, step()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            for x in leaves[:2]:
                x.copy_(torch.randn_like(x, dtype=torch.float32))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("dev", DEVICES)
def test_one_of_two_results_used(dev):
    """No gradient for k' and none asked for the weights."""
    q, k, wq, wk, cos, sin, _, dq, _ = _case(
        dev, torch.float32, 2, 9, 3, 1, 64, 64, False, None, True)
    a, b = (x.detach().requires_grad_(True) for x in (q, k))
    y, _ = OF.qk_norm_rope(a, b, wq, wk, cos, sin)
    ga, gb = torch.autograd.grad(y, (a, b), dq, allow_unused=True)
    y2, _ = OF.qk_norm_rope(a, k, wq, wk, cos, sin)
    assert torch.equal(ga, torch.autograd.grad(y2, a, dq)[0])
    assert gb is None or not bool(gb.any())


@pytest.mark.parametrize("dev", DEVICES)
def test_tables_and_weights_of_any_stride(dev):
    q, k, wq, wk, cos, sin, p, _, _ = _case(
        dev, torch.float32, 2, 9, 3, 1, 64, 64, False, torch.int64, True)
    want = OF.qk_norm_rope(q, k, wq, wk, cos, sin, positions=p)

    def odd(x):  # the same values, every second element of a wider tensor
        return torch.stack([x, torch.zeros_like(x)], -1)[..., 0]

    got = OF.qk_norm_rope(q, k, odd(wq), odd(wk), odd(cos), odd(sin),
                          positions=odd(p))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@gpu
def test_refuses_more_than_a_grid_holds():
    # one token seen many times: no memory is touched
    q = torch.zeros(1, 1, 1, 8, device="cuda").expand(1 << 26, 1, 1, 8)
    w = torch.ones(8, device="cuda")
    with pytest.raises(RuntimeError, match="too many rows"):
        OF.qk_norm_rope(q, q, w, w)
