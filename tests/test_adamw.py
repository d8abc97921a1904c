"""AdamW over flat storage: against the formula in 64 bits, against
torch.optim.AdamW, its 8-bit states, checkpoints and refusals."""
import math

import pytest
import torch

from pytorch_distributed_train_amd.ops import functional as OF
from pytorch_distributed_train_amd.parallel.flat import FlatParams
from pytorch_distributed_train_amd.parallel.optim import FusedAdamW

U = 2.0 ** -24  # half a step of fp32, relative
gpu = pytest.mark.gpu
DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=gpu)]


def _model(seed=1):
    torch.manual_seed(seed)
    return torch.nn.Sequential(
        torch.nn.Linear(9, 17), torch.nn.Tanh(), torch.nn.Linear(17, 3))


def _inputs(n, seed, dev):
    g = torch.Generator().manual_seed(seed)
    p = torch.randn(n, generator=g)
    # magnitudes over nine decades: scales differ from block to block
    mag = 10.0 ** (torch.rand(n // 64, generator=g) * 9 - 8)
    mag = mag.repeat_interleave(64)
    grad = torch.randn(n, generator=g) * mag
    m = torch.randn(n, generator=g) * mag * 0.3
    v = torch.rand(n, generator=g) * mag * mag
    grad[:64] = 0  # a block of nothing
    m[:64] = 0
    v[:64] = 0
    return [x.to(dev) for x in (p, grad, m, v)]


def _oracle(p, g, m, v, t, lr, b1, b2, eps, wd, on):
    """64-bit step; (p, m, v) and the bounds of an fp32 step's error."""
    p, g, m, v = (x.double().cpu() for x in (p, g, m, v))
    on = torch.ones_like(p) if on is None \
        else on.cpu().double().repeat_interleave(64)
    am, av = (b1 * m).abs() + ((1 - b1) * g).abs(), b2 * v + (1 - b2) * g * g
    # b1, 1-b1, the two products and their sum round once each (the inputs'
    # product with grad_scale once more)
    em, ev = 4 * U * am, 6 * U * av
    m, v = b1 * m + (1 - b1) * g, av
    den = (v / (1 - b2 ** t)).sqrt() + eps
    upd = lr / (1 - b1 ** t) * m / den
    keep = p * (1 - lr * wd * on)
    # lr, bc1, quotient, product, sqrt (half of v's error), bc2, product,
    # eps, sum, division: under 16 roundings of the update beside m's own;
    # of p: lr, wd, their product, the difference, the product, the sum
    ep = 16 * U * upd.abs() + lr / (1 - b1 ** t) * em / den \
        + 6 * U * (keep.abs() + p.abs())
    return (keep - upd, m, v), (ep, em, ev)


def _near(got, want, bound, what):
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), \
        f"{what}: off by {float((off - bound).max())} more than allowed"


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("n,t0,wd,part,lr_tensor", [
    (64, 0, 0.0, False, False), (128, 1, 0.01, False, True),
    (64 * 1001, 7, 0.1, True, True), (64 * 40000, 50000, 0.05, True, False)])
def test_step_fp32_states(dev, n, t0, wd, part, lr_tensor):
    p, g, m, v = _inputs(n, n + t0, dev)
    on = None
    if part:
        on = (torch.arange(n // 64) % 3 != 1).to(torch.uint8).to(dev)
    lr, b1, b2, eps = 1e-3, 0.9, 0.95, 1e-8
    # the kernel's lr, betas and scale are fp32 numbers
    lr32 = float(torch.tensor(lr))
    want, bound = _oracle(p, g, m, v, t0 + 1, lr32, b1, b2, eps, wd, on)
    step = torch.full((1,), t0, dtype=torch.int64, device=dev)
    OF.adamw_step(p, g, m, v, step,
                  torch.tensor([lr], device=dev) if lr_tensor else lr32,
                  beta1=b1, beta2=b2, eps=eps, weight_decay=wd, decay=on)
    assert int(step) == t0 + 1
    for x, w, e, what in zip((p, m, v), want, bound, "pmv"):
        _near(x, w, e, what)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("n,t0", [(64, 0), (192, 3), (64 * 1001, 900),
                                  (64 * 40000, 10)])
def test_step_8bit_states(dev, n, t0):
    p, g, m, v = _inputs(n, n + t0 + 5, dev)
    m8, ms = OF.adamw_quantize(m)
    v8, vs = OF.adamw_quantize(v.sqrt(), positive=True)
    lr, b1, b2, eps, wd, gs = 0.0009765625, 0.9, 0.999, 1e-8, 0.01, 0.5
    m0 = m8.cpu().double() * ms.cpu().double().repeat_interleave(64)
    u0 = v8.cpu().double() * vs.cpu().double().repeat_interleave(64)
    (pw, mw, vw), (pe, me, ve) = _oracle(
        p, g * gs, m0, u0 * u0, t0 + 1, lr, b1, b2, eps, wd, None)
    uw = vw.sqrt()
    step = torch.full((1,), t0, dtype=torch.int64, device=dev)
    OF.adamw_step(p, g, m8, v8, step, lr, beta1=b1, beta2=b2, eps=eps,
                  weight_decay=wd, grad_scale=gs, m_scale=ms, v_scale=vs,
                  seed=11)
    # decoding rounds each state twice more (code times scale, its square)
    _near(p, pw, 1.5 * pe, "p")
    tiny = 2.0 ** -100
    for scale, x, e in ((ms, mw, me), (vs, uw, None)):
        top = x.abs().view(-1, 64).amax(1)
        _near(scale, torch.where(top < tiny, 0.0, top / 448),
              top / 448 * 16 * U, "scale")
    ms, vs = (x.cpu().double().repeat_interleave(64) for x in (ms, vs))
    # nearest: half a step, 2^-4 relative, or 2^-10 of the scale below 2^-6
    off = (m8.cpu().double() * ms - mw).abs()
    bound = torch.maximum(mw.abs() * 2.0 ** -4, ms * 2.0 ** -10)
    assert bool((off <= bound * (1 + 2.0 ** -18) + me + tiny).all())
    # at random: a whole step, and above 0 where v is
    got = v8.cpu().double() * vs
    bound = torch.maximum(uw * 2.0 ** -3, vs * 2.0 ** -9)
    assert bool(((got - uw).abs()
                 <= bound * (1 + 2.0 ** -18) + tiny).all())
    live = uw.view(-1, 64).amax(1).repeat_interleave(64) >= 2 * tiny
    assert bool((got[live & (uw > 0)] > 0).all())
    assert bool((got[uw == 0] == 0).all())


@pytest.mark.parametrize("dev", DEVICES)
def test_random_rounding_has_the_values_mean(dev):
    """The stored sqrt(v) is right on average over seeds, so a change below
    half a step is not lost."""
    n, k = 64 * 32, 600
    g0 = torch.Generator().manual_seed(3)
    u = torch.rand(n, generator=g0) + 0.01
    v8, vs = OF.adamw_quantize(u, positive=True)
    u0 = OF.adamw_dequantize(v8, vs).double()
    want = (0.999 * u0 * u0).sqrt()  # no gradient: v shrinks by 0.1%
    total = torch.zeros(n, dtype=torch.float64)
    z = torch.zeros(n, device=dev)
    for s in range(k):
        st = [x.clone().to(dev) for x in (v8, vs)]
        OF.adamw_step(z.clone(), z, z.clone().to(torch.float8_e4m3fn), st[0],
                      torch.full((1,), s, dtype=torch.int64, device=dev),
                      0.0, m_scale=torch.zeros(n // 64, device=dev),
                      v_scale=st[1], seed=1)
        total += OF.adamw_dequantize(*st).double().cpu()
    # one rounding's deviation is at most half a step, u/16; 6 deviations
    # of the mean of k
    dev_ = want / 16 / math.sqrt(k)
    assert bool(((total / k - want).abs() <= 6 * dev_).all())
    # and over all elements the shrinkage is seen
    seen = float((total / k).sum() / u0.sum())
    assert abs(seen - math.sqrt(0.999)) < 6 / 16 / math.sqrt(k * n)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("wd", [0.0, 0.1])
def test_matches_torch_adamw(dev, wd):
    m1, m2 = _model().to(dev), _model().to(dev)
    flat = FlatParams(m1.named_parameters(), device=torch.device(dev))
    ours = FusedAdamW(flat, lr=1e-2, weight_decay=wd)
    ref = torch.optim.AdamW(m2.parameters(), lr=1e-2, weight_decay=wd)
    x = torch.randn(8, 9, generator=torch.Generator().manual_seed(0)).to(dev)
    for i in range(5):
        ours.lr = 1e-2 / (i + 1)
        ref.param_groups[0]["lr"] = 1e-2 / (i + 1)
        ref.zero_grad()
        m2(x).pow(2).mean().backward()
        # the same gradients: only the optimizers are compared
        for a, b in zip(m1.parameters(), m2.parameters()):
            a.grad.copy_(b.grad)
        ours.step()
        ref.step()
        for a, b in zip(m1.parameters(), m2.parameters()):
            # each side within the oracle's bound of some 20 roundings of
            # p + update a step
            assert torch.allclose(a, b, rtol=40 * U * (i + 1),
                                  atol=40 * U * (i + 1) * 1e-1)
    ours.load_state_dict(ref.state_dict() | {"state": {
        i: ref.state_dict()["state"][flat.num_params - 1 - i]
        for i in range(flat.num_params)}})
    off, n = flat.offsets[0], flat.sizes[0]
    assert torch.equal(ours.exp_avg[off:off + n].cpu(),
                       ref.state_dict()["state"][flat.num_params - 1]
                       ["exp_avg"].reshape(-1).cpu())
    assert int(ours.step_count) == 5


def _flat_grads(flat, seed):
    g = torch.Generator().manual_seed(seed)
    for i in range(flat.num_params):
        flat.grad_view(i).copy_(torch.randn(flat.shapes[i], generator=g))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("bits2", [8, 32])
def test_state_dict_roundtrip(bits, bits2):
    flat = FlatParams(_model().named_parameters())
    opt = FusedAdamW(flat, lr=0.1, state_bits=bits)
    for s in range(3):
        _flat_grads(flat, s)
        opt.step()
    sd = opt.state_dict()
    assert list(sd["state"][0])[:3] == ["step", "exp_avg", "exp_avg_sq"]
    flat2 = FlatParams(_model().named_parameters())
    flat2.master.copy_(flat.master)
    opt2 = FusedAdamW(flat2, lr=0.5, state_bits=bits2)
    opt2.load_state_dict(sd)
    assert opt2.lr == 0.1 and int(opt2.step_count) == 3
    if bits == bits2:
        assert torch.equal(opt.exp_avg.float(), opt2.exp_avg.float())
        assert torch.equal(opt.exp_avg_sq.float(), opt2.exp_avg_sq.float())
        _flat_grads(flat, 9)
        flat2.grad.copy_(flat.grad)
        opt.step()
        opt2.step()
        assert torch.equal(flat.master, flat2.master)
        return

    def wide(o, key, scale):
        x = getattr(o, key).float()
        if o.state_bits == 8:
            x = OF.adamw_dequantize(getattr(o, key), getattr(o, scale))
            x = x * x if key == "exp_avg_sq" else x
        return x

    for key in ("exp_avg", "exp_avg_sq"):
        a = wide(opt, key, key + "_scale")
        b = wide(opt2, key, key + "_scale")
        # half a step of e4m3, twice that in the square; the least values of
        # a block as far as half of e4m3's least step over 448
        rel = (1 + 2.0 ** -4) ** 2 - 1 if key == "exp_avg_sq" else 2.0 ** -4
        top = a.abs().max()
        assert bool(((a - b).abs() <= rel * 1.0001 * a.abs()
                     + top * 2.0 ** -9 / 448).all()), key


def test_decay_only_where_asked():
    flat = FlatParams(_model().named_parameters())
    before = flat.master.clone()
    opt = FusedAdamW(flat, lr=0.1, weight_decay=0.5,
                     decay=lambda name, shape: len(shape) > 1)
    opt.step()  # no gradient: decay alone
    for i in range(flat.num_params):
        off, n = flat.offsets[i], flat.sizes[i]
        k = 0.95 if len(flat.shapes[i]) > 1 else 1.0
        assert torch.allclose(flat.master[off:off + n],
                              before[off:off + n] * k, rtol=4 * U, atol=0)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_gradient_not_finite_shows(dev, bad):
    p, g, m, v = _inputs(256, 1, dev)
    m8, ms = OF.adamw_quantize(m)
    v8, vs = OF.adamw_quantize(v.sqrt(), positive=True)
    g[70] = bad
    step = torch.zeros(1, dtype=torch.int64, device=dev)
    OF.adamw_step(p, g, m8, v8, step, 0.1, m_scale=ms, v_scale=vs)
    assert bool(torch.isnan(p[70]))
    fine = torch.ones(256, dtype=torch.bool)
    fine[70] = False
    assert bool(torch.isfinite(p.cpu()[fine]).all())
    wide = OF.adamw_dequantize(v8, vs).cpu()
    assert not bool(torch.isfinite(wide[70]))
    assert bool(torch.isfinite(wide[128:]).all())


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    def call(**kw):
        n = kw.pop("n", 128)
        a = {"p": torch.zeros(n, device=dev), "g": torch.zeros(n, device=dev),
             "m": torch.zeros(n, device=dev), "v": torch.zeros(n, device=dev),
             "step": torch.zeros(1, dtype=torch.int64, device=dev),
             "lr": 0.1}
        a.update(kw)
        with pytest.raises((ValueError, RuntimeError)):
            OF.adamw_step(**a)

    def z(n, dt=torch.float32):
        return torch.zeros(n, device=dev).to(dt)

    call(n=100)
    call(g=z(64))
    call(m=z(128, torch.float16))
    call(m=z(256)[::2])
    call(m_scale=z(2))
    call(m_scale=z(2), v_scale=z(2))  # fp32 states beside scales
    call(m=z(128, torch.float8_e4m3fn), v=z(128, torch.float8_e4m3fn))
    call(m=z(128, torch.float8_e4m3fn), v=z(128, torch.float8_e4m3fn),
         m_scale=z(2), v_scale=z(1))
    call(decay=z(1, torch.uint8))
    call(decay=z(2))
    call(step=z(1))
    call(beta2=1.0)
    call(beta1=-0.1)
    call(eps=-1.0)
    flat = FlatParams(_model().named_parameters())
    with pytest.raises(ValueError):
        FusedAdamW(flat, lr=0.1, state_bits=4)
    with pytest.raises(ValueError):
        FusedAdamW(flat, lr=0.1, betas=(0.9, 1.0))


@pytest.mark.parametrize("dev", DEVICES)
def test_empty(dev):
    z = torch.zeros(0, device=dev)
    step = torch.zeros(1, dtype=torch.int64, device=dev)
    OF.adamw_step(z, z, z, z, step, 0.1)
    assert int(step) == 1


def test_load_state_dict_replaces_and_refuses():
    from pytorch_distributed_train_amd.parallel.optim import FusedSGD
    flat = FlatParams(_model().named_parameters())
    for bits in (8, 32):
        opt = FusedAdamW(flat, lr=0.1, state_bits=bits)
        _flat_grads(flat, 1)
        opt.step()
        sd = opt.state_dict()
        opt.step()
        only = {**sd, "state": {0: sd["state"][0]}}
        opt.load_state_dict(only)
        assert int(opt.step_count) == 1
        off = flat.offsets[1]
        assert not bool(opt.exp_avg[off:].float().any())
        assert bool(opt.exp_avg[:off].float().any())
        opt.load_state_dict({**sd, "state": {}})
        assert int(opt.step_count) == 0
        assert not bool(opt.exp_avg_sq.float().any())
        with pytest.raises(ValueError):
            opt.load_state_dict({**sd, "state": {99: sd["state"][0]}})
        with pytest.raises(ValueError):
            opt.load_state_dict(FusedSGD(flat, 0.1, 0.9).state_dict())


def test_ranks_stay_alike_with_8bit_states(tmp_path):
    """The random rounding is the same on every rank."""
    from test_ddp_gloo import _run_workers
    _run_workers(False, False, tmp_path,
                 ("--optimizer", "adamw", "--adam-bits", "8", "--lr",
                  "0.001"))
    a, b = (torch.load(str(tmp_path / f"rank{r}.pt"), weights_only=True)
            for r in range(2))
    assert torch.equal(a["grad"], b["grad"])
    assert torch.equal(a["master"], b["master"])


@gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_captured_step_replays_as_the_next(bits):
    """Replays advance the step number and follow the learning rate, as
    eager steps do, with eager work between them."""
    def make():
        m = _model().to("cuda")
        flat = FlatParams(m.named_parameters(), device=torch.device("cuda"))
        return flat, FusedAdamW(flat, lr=0.01, state_bits=bits, seed=5)

    (fa, a), (fb, b) = make(), make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _flat_grads(fa, 0)
        a.step()
    torch.cuda.current_stream().wait_stream(side)
    _flat_grads(fb, 0)
    b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for i in range(4):
        for f, o in ((fa, a), (fb, b)):
            _flat_grads(f, i + 1)
            o.lr = 0.01 / (i + 1)
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        assert torch.equal(fa.master, fb.master), i
        assert torch.equal(a.exp_avg_sq.float(), b.exp_avg_sq.float()), i
        assert int(a.step_count) == int(b.step_count) == i + 2


@gpu
def test_kernel_and_plain_path_agree():
    """The same random bits on both devices: the codes of sqrt(v) differ
    only where its own rounding error crosses a border."""
    n = 64 * 500
    p, g, m, v = _inputs(n, 77, "cpu")
    out = []
    for dev in ("cpu", "cuda"):
        m8, ms = OF.adamw_quantize(m)
        v8, vs = OF.adamw_quantize(v.sqrt(), positive=True)
        a = [x.clone().to(dev) for x in (p, g, m8, v8, ms, vs)]
        OF.adamw_step(a[0], a[1], a[2], a[3],
                      torch.full((1,), 41, dtype=torch.int64, device=dev),
                      0.01, m_scale=a[4], v_scale=a[5], seed=123)
        out.append([x.float().cpu() for x in a])
    for i, what in ((2, "m"), (3, "sqrt(v)")):
        differ = (out[0][i] != out[1][i]).float().mean()
        # a few roundings, 2^-22 of a value, against steps of 2^-4: one
        # element in 2^18 at the most is expected to cross
        assert float(differ) <= 1e-3, what
