"""The operators together, as training uses them: the ViT's attention with
normed and rotated queries and keys, AdamW, the training command."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import train as train_mod  # repo-root entrypoint
from pytorch_distributed_train_amd.models import build_model
from pytorch_distributed_train_amd.models.vit import MultiheadSelfAttention
from pytorch_distributed_train_amd.ops import functional as OF

gpu = pytest.mark.gpu


def _attention64(m, x, h):
    """The module's function in 64 bits, from its parameters."""
    p = {n: t.detach().double().cpu().requires_grad_(True)
         for n, t in m.named_parameters()}
    b, s, d = x.shape
    hd = d // h
    x = x.detach().double().cpu().requires_grad_(True)
    qkv = x @ p["in_proj_weight"].t() + p["in_proj_bias"]
    q, k, v = qkv.view(b, s, 3, h, hd).permute(2, 0, 3, 1, 4)

    def prep(t, w):
        t = t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
        side = math.isqrt(s - 1)
        f = 100.0 ** (-torch.arange(0, hd // 2, 2, dtype=torch.float64)
                      / (hd // 2))
        at = torch.arange(side * side)
        a = torch.cat([(at // side)[:, None] * f, (at % side)[:, None] * f],
                      1)
        a = torch.cat([torch.zeros(1, hd // 2, dtype=a.dtype), a])
        z = torch.complex(t[..., :hd // 2], t[..., hd // 2:]) \
            * torch.polar(torch.ones_like(a), a)
        return torch.cat([z.real, z.imag], -1)

    q, k = prep(q, p["q_norm_weight"]), prep(k, p["k_norm_weight"])
    o = torch.softmax(q @ k.transpose(-1, -2) / hd ** 0.5, -1) @ v
    o = o.permute(0, 2, 1, 3).reshape(b, s, d)
    return x, p, o @ p["out_proj.weight"].t() + p["out_proj.bias"]


def _module(d, h):
    torch.manual_seed(1)
    m = MultiheadSelfAttention(d, h, qk_norm_rope=True)
    with torch.no_grad():
        m.q_norm_weight.uniform_(0.5, 1.5)
        m.k_norm_weight.uniform_(0.5, 1.5)
        m.in_proj_bias.normal_()
    return m


@pytest.mark.parametrize("dev,dtype,tol", [
    # under 100 roundings of 2^-24 in a row
    ("cpu", torch.float32, 100 * 2.0 ** -24),
    # x, the weights, qkv, q and k, P, out, the projection, and their
    # gradients' counterparts: 14 roundings of at most 2^-8, by the norms
    pytest.param("cuda", torch.bfloat16, 14 * 2.0 ** -8, marks=gpu),
    pytest.param("cuda", torch.float16, 14 * 2.0 ** -11, marks=gpu)])
def test_attention_module(dev, dtype, tol):
    b, s, d, h = 3, 50, 128, 2
    m = _module(d, h).to(dev)
    x = torch.randn(b, s, d).to(dtype).to(dev).requires_grad_(True)
    y = m(x)
    g = torch.randn(b, s, d).to(dtype).to(dev)
    y.backward(g)
    x64, p64, y64 = _attention64(m, x, h)
    y64.backward(g.double().cpu())

    def near(a, w, what):
        off = float((a.double().cpu() - w).norm() / w.norm())
        assert off <= tol, f"{what}: {off} > {tol}"

    near(y.detach(), y64.detach(), "y")
    near(x.grad, x64.grad, "dx")
    for n, t in m.named_parameters():
        near(t.grad, p64[n].grad, n)


def test_rotation_sees_differences_of_positions_only():
    cos, sin = OF.rope_tables_2d(5, 6, 16, prefix=1)
    assert cos.shape == (31, 8)
    assert bool((cos[0] == 1).all()) and bool((sin[0] == 0).all())
    q, k = torch.randn(2, 16, dtype=torch.float64)

    def score(a, b):  # the same q and k at grid places a and b
        at = torch.tensor([[1 + a[0] * 6 + a[1], 1 + b[0] * 6 + b[1]]])
        x, y = OF.qk_norm_rope(q.view(1, 1, 1, 16).expand(1, 2, 1, 16),
                               k.view(1, 1, 1, 16).expand(1, 2, 1, 16),
                               None, None, cos.double(), sin.double(),
                               positions=at)
        return float(x[0, 0, 0] @ y[0, 1, 0])

    # tables of 32 bits: angles off by 2^-24 of a turn's sine at the most
    assert abs(score((0, 1), (2, 4)) - score((2, 2), (4, 5))) < 1e-5
    assert abs(score((0, 1), (2, 4)) - score((0, 1), (2, 3))) > 1e-3


def test_model_and_refusals():
    with pytest.raises(ValueError):
        build_model("resnet18", 10, torch.float32, qk_norm_rope=True)
    m = MultiheadSelfAttention(32, 2, qk_norm_rope=True)
    with pytest.raises(ValueError):
        m(torch.zeros(1, 7, 32))  # no square grid and class token
    with pytest.raises(ValueError):
        m(torch.zeros(1, 5, 32), nvalid=4)
    plain = MultiheadSelfAttention(32, 2)
    assert not any("norm" in n for n in plain.state_dict())
    assert set(m.state_dict()) - set(plain.state_dict()) \
        == {"q_norm_weight", "k_norm_weight"}


def _argv(tmp_path, *extra):
    return ["--model", "resnet18", "--data", "synthetic-cifar10", "--dtype",
            "fp32", "--device", "cpu", "--batch-size", "4", "--num-samples",
            "8", "--epochs", "2", "--lr", "0.001", "--checkpoint-dir",
            str(tmp_path), "--checkpoint-freq", "1", "--optimizer", "adamw",
            "--no-decay-1d", *extra]


@pytest.mark.parametrize("bits", ["32", "8"])
def test_train_command_with_adamw(tmp_path, monkeypatch, bits):
    monkeypatch.delenv("RANK", raising=False)
    monkeypatch.delenv("WORLD_SIZE", raising=False)
    argv = _argv(tmp_path, "--adam-bits", bits)
    assert train_mod.main(argv) == 0
    ckpt = tmp_path / "resnet18_checkpoint.pt"
    sd = torch.load(str(ckpt), weights_only=False)["optimizer"]
    assert int(sd["state"][0]["step"]) == 4  # 2 epochs of 2 steps
    assert ("exp_avg_scale" in sd["state"][0]) == (bits == "8")
    assert train_mod.main([*argv, "--resume", str(ckpt), "--epochs",
                           "3"]) == 0
    sd = torch.load(str(ckpt), weights_only=False)["optimizer"]
    assert int(sd["state"][0]["step"]) == 6


def _trainer(**kw):
    from pytorch_distributed_train_amd.engine import Trainer
    from pytorch_distributed_train_amd.flags import DistEnv, build_parser
    args = build_parser().parse_args([
        "--model", "vit_b_16", "--dtype", "bf16", "--qk-norm-rope",
        "--optimizer", "adamw", "--adam-bits", "8", "--no-decay-1d",
        "--lr", "0.0003", "--weight-decay", "0.05"])
    return Trainer(args, DistEnv())


@gpu
def test_trainer_steps_eager_and_captured():
    """An eager step, three warm-up steps and four replays do what eight
    eager steps do, with eager work between the replays."""
    x = torch.randn(4, 3, 224, 224, device="cuda")
    y = torch.randint(0, 1000, (4,), device="cuda")
    a, b = _trainer(), _trainer()
    for t in (a, b):
        t.model.train()
        t.train_step(x, y)
    assert a.enable_hip_graph(x, y)
    for _ in range(3):
        b.train_step(x, y)
    for i in range(4):
        for t in (a, b):
            t.optimizer.lr = 3e-4 / (i + 1)
        la = a.graph_step(x, y).clone()
        lb = b.train_step(x, y)
        torch.cuda.synchronize()
        assert math.isfinite(float(la))
        assert torch.equal(la, lb), (i, float(la), float(lb))
        assert torch.equal(a.flat.master, b.flat.master), i
    names = [n for n in a.flat.names if "norm_weight" in n]
    assert len(names) == 24
    for i, n in enumerate(a.flat.names):
        assert float(a.flat.grad_view(i).abs().max()) > 0.0 \
            or n.endswith("class_token"), n
