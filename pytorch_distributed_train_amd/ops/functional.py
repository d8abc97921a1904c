"""Autograd ops over NHWC activations.

Every op has two implementations:
  - CUDA (ROCm) tensors -> the in-tree gfx950 HIP extension (backend.ext()),
    which raises loudly if not built — no silent eager fallback on GPU;
  - CPU tensors -> a plain PyTorch fp32 reference. This is the numerics
    oracle the GPU kernels are tested against (tests/test_kernels_gpu.py)
    and what the gloo world_size=2 CPU plumbing config runs on.

Layout contract: activations are [N, H, W, C] contiguous ("NHWC"); C is
innermost so channel vectors are contiguous for MFMA K-dim staging and BN
reductions. Conv weights: master fp32 [K, C, R, S] (torch checkpoint layout,
SURVEY.md §5.4 checkpoint parity), packed compute copy [R, S, C, K] in the
compute dtype. Linear weights: master fp32 [N, K] (torch layout), packed =
same layout cast to the compute dtype (the MFMA GEMM consumes B^T = [N, K]).

Reference behavior being rebuilt: MIOpen conv, ATen
batch_norm kernels, fused log-softmax+NLL, maxpool/avgpool — re-designed
as CDNA4 kernels, not ported.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from .backend import ext


def _nhwc_to_nchw(x):
    return x.permute(0, 3, 1, 2).contiguous()


def _nchw_to_nhwc(x):
    return x.permute(0, 2, 3, 1).contiguous()


def conv_out_dim(h: int, k: int, stride: int, pad: int) -> int:
    return (h + 2 * pad - k) // stride + 1


# ---------------------------------------------------------------------------
# Convolution (implicit GEMM on GPU)
# ---------------------------------------------------------------------------

class GradHolder:
    """Per-block, per-iteration slot carrying the residual-path gradient
    (GradHolder protocol): the producer Function (the block's
    last BN `dres`, or the downsample conv's `dx`) stores the tensor here
    and returns None to autograd — no fork add exists; the consumer (the
    PREVIOUS block's BN backward) sums it as a second dy inside its
    reduce/elemt kernels and clears the slot. A slot found still-full at
    the next forward means the fold never happened, and the block raises.
    Pure python; the tensors it references are ordinary stream-ordered
    outputs, so this works in eager mode and under hipGraph capture."""
    __slots__ = ("t",)

    def __init__(self):
        self.t = None


def fork_fuse_enabled() -> bool:
    import os
    return not os.environ.get("PDTA_NO_FORK_FUSE")


class Conv2dNHWC(torch.autograd.Function):
    """y[n,p,q,k] = sum_{r,s,c} x[n, p*st-pad+r, q*st-pad+s, c] * w[k,c,r,s].

    GPU: implicit-GEMM MFMA kernels (csrc/conv.hip). Two compute-dtype
    weight packs keep every direction K-contiguous ("nt"-shaped):
      wt [K,R,S,C] for forward, w2 [R,S,C,K] for backward-data (see
      conv.hip header). Gradient is returned for the master fp32 weight
    directly in its [K,C,R,S] layout (the wrw kernel scatters there).
    """

    @staticmethod
    def forward(ctx, x, weight, wt, w2, stride: int, pad: int,
                want_bn_stats: bool = False, dx_sink=None, gslot=None):
        ctx.stride, ctx.pad = stride, pad
        ctx.dx_sink = dx_sink
        ctx.gslot = gslot  # (grad_view, notify) direct-grad destination
        # the bn-stats `part` output is non-differentiable; without this,
        # autograd MATERIALIZES a zero gradient for it every backward
        # (measured: ~53 FillFunctor launches/step on ResNet-50)
        ctx.set_materialize_grads(False)
        if x.is_cuda:
            # stem (C % 64 != 0): cache the im2col image for bwd-weight.
            # NOTE grad mode is always DISABLED inside a custom Function's
            # forward, so gate on the weight's requires_grad instead (a
            # torch.is_grad_enabled() gate here is always False — measured
            # as a full extra im2col pass per step)
            want_xcol = x.shape[3] % 64 != 0 and weight.requires_grad
            out = ext().conv2d_fwd(x, wt, stride, pad, want_bn_stats,
                                   want_xcol)
            xcol = out[-1] if want_xcol else None
            ctx.save_for_backward(x, weight, w2, xcol)
            if want_bn_stats:
                y, part = out[0], out[1]
                ctx.mark_non_differentiable(part)
                return y, part
            return out[0]
        ctx.save_for_backward(x, weight, w2, None)
        # CPU reference (fp32)
        w = weight.float()
        y = F.conv2d(_nhwc_to_nchw(x).float(), w, stride=stride, padding=pad)
        return _nchw_to_nhwc(y).to(x.dtype)

    @staticmethod
    def backward(ctx, dy, _dpart=None):
        x, weight, w2, xcol = ctx.saved_tensors
        stride, pad = ctx.stride, ctx.pad
        dy = dy.contiguous()
        need_dx = ctx.needs_input_grad[0]
        need_dw = ctx.needs_input_grad[1]
        dx = dw = None
        if x.is_cuda:
            if need_dx:
                dx = ext().conv2d_bwd_data(dy, w2, x.shape[1], x.shape[2],
                                           stride, pad)
                if ctx.dx_sink is not None:
                    # residual-path producer (GradHolder protocol): the
                    # previous block's BN backward reads this as its
                    # second dy; autograd sees None — no fork add exists
                    ctx.dx_sink.t = dx
                    dx = None
            if need_dw:
                if ctx.gslot is not None:
                    # direct-grad: write straight into the flat slice and
                    # return None (no AccumulateGrad add); tell the
                    # reducer the param arrived
                    view, notify = ctx.gslot
                    ext().conv2d_bwd_weight(x, dy, weight.shape[2],
                                            weight.shape[3], stride, pad,
                                            xcol_cached=xcol, out=view)
                    if notify is not None:
                        notify()
                    dw = None
                else:
                    dw = ext().conv2d_bwd_weight(x, dy, weight.shape[2],
                                                 weight.shape[3], stride,
                                                 pad, xcol_cached=xcol)
        else:
            x_nchw = _nhwc_to_nchw(x).float()
            dy_nchw = _nhwc_to_nchw(dy).float()
            w = weight.float()
            if need_dx:
                dx = torch.nn.grad.conv2d_input(x_nchw.shape, w, dy_nchw,
                                                stride=stride, padding=pad)
                dx = _nchw_to_nhwc(dx).to(x.dtype)
            if need_dw:
                dw = torch.nn.grad.conv2d_weight(x_nchw, w.shape, dy_nchw,
                                                 stride=stride, padding=pad)
        return dx, dw, None, None, None, None, None, None, None


def conv2d_nhwc(x, weight, wt, w2, stride: int = 1, pad: int = 0,
                want_bn_stats: bool = False, dx_sink=None, gslot=None):
    if want_bn_stats or dx_sink is not None or gslot is not None:
        return Conv2dNHWC.apply(x, weight, wt, w2, stride, pad,
                                want_bn_stats, dx_sink, gslot)
    return Conv2dNHWC.apply(x, weight, wt, w2, stride, pad)


# ---------------------------------------------------------------------------
# BatchNorm (+ fused ReLU)
# ---------------------------------------------------------------------------

def _bn_cpu_stats(x):
    x32 = x.float()
    n = x.shape[0] * x.shape[1] * x.shape[2]
    mean = x32.sum(dim=(0, 1, 2)) / n
    var = x32.pow(2).sum(dim=(0, 1, 2)) / n - mean * mean
    return mean, var.clamp_(min=0.0)


class BatchNorm2dNHWCFn(torch.autograd.Function):
    """Training-mode BN over [N,H,W,C] with optional fused ReLU.

    Decomposed exactly as the kernels are (stats -> apply; bwd_reduce ->
    bwd_elemt) so SyncBatchNorm reuses the same kernels with an all-gather
    between stats and apply.
    """

    @staticmethod
    def forward(ctx, x, weight, bias, mean, invstd, fuse_relu: bool,
                comm=None, count_override=None, residual=None,
                dres_sink=None, dy2_source=None, gslot_w=None,
                gslot_b=None):
        # mean/invstd are per-channel fp32, computed by the module (local
        # stats for BN, cross-rank combined for SyncBN). For SyncBN, `comm`
        # all-reduces the backward sums and `count_override` is the GLOBAL
        # element count (all_reduce of [sum_dy, sum_dy_xmu]).
        # `residual` fuses the ResNet join: y = relu(bn(x) + residual) in
        # one pass (requires fuse_relu).
        mask = None
        if x.is_cuda:
            import os as _os
            if fuse_relu and residual is not None \
                    and _os.environ.get("PDTA_BN_BITMASK"):
                # 1-bit join relu mask: NEGATIVE result at B=256 (-2%
                # step: the byte loads are 8x redundant across lanes and
                # the emit costs more than the saved y pass) — kept
                # opt-in for re-evaluation at other shapes
                y, mask = ext().bn_apply_v(x, weight, bias, mean, invstd,
                                           fuse_relu, residual, True)
            else:
                y = ext().bn_apply(x, weight, bias, mean, invstd,
                                   fuse_relu, residual)
        else:
            x32 = x.float()
            xhat = (x32 - mean) * invstd
            y = xhat * weight.float() + bias.float()
            if residual is not None:
                y = y + residual.float()
            if fuse_relu:
                y = y.clamp_(min=0.0)
            y = y.to(x.dtype)
        ctx.fuse_relu = fuse_relu
        ctx.comm = comm
        ctx.count_override = count_override
        ctx.has_residual = residual is not None
        ctx.dres_sink = dres_sink
        ctx.dy2_source = dy2_source
        ctx.gslot_w, ctx.gslot_b = gslot_w, gslot_b
        ctx.save_for_backward(x, weight, bias, mean, invstd, y, mask)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, bias, mean, invstd, y, mask = ctx.saved_tensors
        fuse_relu = ctx.fuse_relu
        dy = dy.contiguous()
        dy2 = None
        if ctx.dy2_source is not None and ctx.dy2_source.t is not None:
            # second incoming gradient (next block's residual path),
            # summed in-kernel (two-dy backward)
            dy2 = ctx.dy2_source.t
            ctx.dy2_source.t = None
        n = x.shape[0] * x.shape[1] * x.shape[2]
        if ctx.count_override is not None:
            n = ctx.count_override
        dres = None
        if x.is_cuda:
            # ReLU mask: residual joins must read the stored relu output
            # (pre-activation includes the identity branch); plain conv->
            # bn->relu recomputes the mask from xhat in-kernel and never
            # re-reads y (one whole HBM pass saved per kernel)
            relu_y = y if (fuse_relu and ctx.has_residual) else None
            premask = fuse_relu and not ctx.has_residual
            # direct-grad: dbias == sum_dy — have the finalize kernel
            # write it straight into the flat slice (no D2D copy); with a
            # comm the slice still holds the LOCAL sums (correct: DDP
            # averages param grads) and the packed allreduce reads it
            b_view = ctx.gslot_b[0] if ctx.gslot_b is not None else None
            red = ext().bn_bwd_reduce(
                x, dy, relu_y if mask is None else None, mean,
                invstd=invstd if premask else None,
                weight=weight if premask else None,
                bias=bias if premask else None, dy2=dy2, mbits=mask,
                sum_dy_out=b_view)
            sum_dy, sum_dy_xmu = red[0], red[1]
            dy_comb = None
            if dy2 is not None:
                # two-dy: the reduce pass wrote the masked combined dy;
                # the elemt pass now runs mask-free on that one tensor,
                # and it IS the residual-path gradient (dres)
                dy_comb = red[2]
            # param grads from LOCAL sums (DDP averages them afterwards,
            # matching torch SyncBN's split of responsibilities)
            if ctx.gslot_w is not None and x.is_cuda:
                torch.mul(sum_dy_xmu, invstd, out=ctx.gslot_w[0])
                if ctx.gslot_w[1] is not None:
                    ctx.gslot_w[1]()
                dweight = None
            else:
                dweight = sum_dy_xmu * invstd
            if ctx.gslot_b is not None and x.is_cuda:
                # sum_dy IS the flat slice (written by the reduce)
                if ctx.gslot_b[1] is not None:
                    ctx.gslot_b[1]()
                dbias = None
            else:
                dbias = sum_dy.clone() if ctx.comm is not None else sum_dy
            if ctx.comm is not None:
                # [sum_dy ‖ sum_dy_xmu ‖ local_count] in ONE all-reduce;
                # normalizing by the reduced count on-device keeps the
                # path host-sync-free AND exact for ragged rank batches
                # (fused pack/div kernels: no cat/full/slice launches)
                c = sum_dy.numel()
                local_n = float(x.shape[0] * x.shape[1] * x.shape[2])
                packed = ext().syncbn_pack2(sum_dy, sum_dy_xmu, local_n)
                ctx.comm.allreduce_sum(packed).sync_stream()
                ext().syncbn_div(packed, c)
                sum_dy, sum_dy_xmu = packed[:c], packed[c:2 * c]
                n = 1.0
            if dy_comb is not None:
                out = ext().bn_bwd_elemt(x, dy_comb, None, mean, invstd,
                                         weight, sum_dy.contiguous(),
                                         sum_dy_xmu.contiguous(), float(n),
                                         False)
                dx = out[0]
                dres = dy_comb if ctx.has_residual else None
            else:
                out = ext().bn_bwd_elemt(x, dy, relu_y, mean, invstd,
                                         weight, sum_dy.contiguous(),
                                         sum_dy_xmu.contiguous(), float(n),
                                         ctx.has_residual,
                                         bias=bias if premask else None)
                dx = out[0]
                if ctx.has_residual:
                    dres = out[1]
            if dres is not None and ctx.dres_sink is not None:
                # residual-path producer (GradHolder protocol): the
                # consumer BN sums this as its second dy; autograd
                # sees None
                ctx.dres_sink.t = dres
                dres = None
        else:
            dy32 = dy.float()
            if dy2 is not None:
                dy32 = dy32 + dy2.float()
            if fuse_relu:
                dy32 = dy32 * (y.float() > 0)
            x32 = x.float()
            xmu = x32 - mean
            sum_dy = dy32.sum(dim=(0, 1, 2))
            sum_dy_xmu = (dy32 * xmu).sum(dim=(0, 1, 2))
            dweight = sum_dy_xmu * invstd
            dbias = sum_dy.clone() if ctx.comm is not None else sum_dy
            if ctx.comm is not None:
                c = sum_dy.numel()
                local_n = float(x.shape[0] * x.shape[1] * x.shape[2])
                packed = torch.cat([sum_dy, sum_dy_xmu,
                                    torch.full((1,), local_n,
                                               dtype=torch.float32)])
                ctx.comm.allreduce_sum(packed).wait()
                packed[:2 * c] /= packed[2 * c]
                sum_dy, sum_dy_xmu = packed[:c], packed[c:2 * c]
                n = 1.0
            w32 = weight.float()
            if ctx.has_residual:
                dres = dy32.to(x.dtype)
            dx = (dy32 - sum_dy / n - xmu * invstd * invstd * sum_dy_xmu / n)
            dx = (dx * w32 * invstd).to(x.dtype)
        return (dx, dweight, dbias, None, None, None, None, None,
                dres, None, None, None, None)


def bn_stats(x):
    """Per-channel (mean, var) over N*H*W in fp32. GPU: reduction kernel,
    or finalize-only when the producing conv pre-reduced the partials."""
    if x.is_cuda:
        part = getattr(x, "_pdta_bn_part", None)
        if part is not None:
            rows = x.shape[0] * x.shape[1] * x.shape[2]
            return ext().bn_stats_from_part(part, rows, x.shape[3])
        return ext().bn_stats(x)
    return _bn_cpu_stats(x)


def bn_stats_train(x, running_mean, running_var, momentum, eps):
    """(mean, invstd) + in-kernel running-stat update — GPU training fast
    path (one kernel pair instead of stats + 4 python-side buffer ops)."""
    return ext().bn_stats_train(x, running_mean, running_var, momentum, eps)


def bn_stats_train_from_part(part, rows, running_mean, running_var,
                             momentum, eps):
    """(mean, invstd) finalized from a conv2d_nhwc(want_bn_stats=True)
    partial slab — the stage-1 pass over the activation never runs."""
    return ext().bn_stats_train_from_part(part, rows, running_mean,
                                          running_var, momentum, eps)


def bn_train(x, weight, bias, mean, invstd, fuse_relu=False, comm=None,
             count=None, residual=None, dres_sink=None, dy2_source=None,
             gslot_w=None, gslot_b=None):
    return BatchNorm2dNHWCFn.apply(x, weight, bias, mean, invstd, fuse_relu,
                                   comm, count, residual, dres_sink,
                                   dy2_source, gslot_w, gslot_b)


def bn_infer(x, weight, bias, running_mean, running_var, eps, fuse_relu=False,
             residual=None):
    invstd = (running_var.float() + eps).rsqrt()
    if x.is_cuda:
        return ext().bn_apply(x, weight, bias, running_mean.float(), invstd,
                              fuse_relu, residual)
    x32 = x.float()
    y = (x32 - running_mean) * invstd * weight.float() + bias.float()
    if residual is not None:
        y = y + residual.float()
    if fuse_relu:
        y = y.clamp_(min=0.0)
    return y.to(x.dtype)


# ---------------------------------------------------------------------------
# Elementwise: relu, residual add+relu
# ---------------------------------------------------------------------------

class ReLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        y = ext().relu_fwd(x) if x.is_cuda else x.clamp(min=0)
        ctx.save_for_backward(y)
        return y

    @staticmethod
    def backward(ctx, dy):
        (y,) = ctx.saved_tensors
        if y.is_cuda:
            return ext().relu_bwd_mask(dy.contiguous(), y)
        return dy * (y > 0)


class AddReLU(torch.autograd.Function):
    """y = relu(a + b) — the residual join, one kernel instead of two."""

    @staticmethod
    def forward(ctx, a, b):
        if a.is_cuda:
            y = ext().add_relu_fwd(a, b)
        else:
            y = (a + b).clamp_(min=0)
        ctx.save_for_backward(y)
        return y

    @staticmethod
    def backward(ctx, dy):
        (y,) = ctx.saved_tensors
        if y.is_cuda:
            d = ext().relu_bwd_mask(dy.contiguous(), y)
        else:
            d = dy * (y > 0)
        return d, d


def relu(x):
    return ReLU.apply(x)


def add_relu(a, b):
    return AddReLU.apply(a, b)


# ---------------------------------------------------------------------------
# Pooling
# ---------------------------------------------------------------------------

class MaxPool2dNHWC(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kernel: int, stride: int, pad: int):
        ctx.kernel, ctx.stride, ctx.pad = kernel, stride, pad
        ctx.in_shape = x.shape
        if x.is_cuda:
            y, idx = ext().maxpool_fwd(x, kernel, stride, pad)
            ctx.save_for_backward(idx)
            ctx.gpu = True
            return y
        x_nchw = _nhwc_to_nchw(x).float()
        y, idx = F.max_pool2d(x_nchw, kernel, stride, pad, return_indices=True)
        ctx.save_for_backward(idx)
        ctx.gpu = False
        return _nchw_to_nhwc(y).to(x.dtype)

    @staticmethod
    def backward(ctx, dy):
        (idx,) = ctx.saved_tensors
        n, h, w, c = ctx.in_shape
        dy = dy.contiguous()
        if ctx.gpu:
            dx = ext().maxpool_bwd(dy, idx, h, w, ctx.kernel, ctx.stride,
                                   ctx.pad)
            return dx, None, None, None
        dy_nchw = _nhwc_to_nchw(dy).float()
        # scatter_ADD (not max_unpool, which overwrites duplicate winners of
        # overlapping windows) to match true max_pool backward semantics
        nn_, cc = dy_nchw.shape[0], dy_nchw.shape[1]
        dx = torch.zeros(nn_, cc, h * w, dtype=dy_nchw.dtype)
        dx.scatter_add_(2, idx.view(nn_, cc, -1), dy_nchw.view(nn_, cc, -1))
        dx = dx.view(nn_, cc, h, w)
        return _nchw_to_nhwc(dx).to(dy.dtype), None, None, None


class GlobalAvgPoolNHWC(torch.autograd.Function):
    """[N,H,W,C] -> [N,C] mean over H,W."""

    @staticmethod
    def forward(ctx, x):
        ctx.in_shape = x.shape
        if x.is_cuda:
            return ext().avgpool_global_fwd(x)
        return x.float().mean(dim=(1, 2)).to(x.dtype)

    @staticmethod
    def backward(ctx, dy):
        n, h, w, c = ctx.in_shape
        dy = dy.contiguous()
        if dy.is_cuda:
            return ext().avgpool_global_bwd(dy, h, w)
        dx = (dy.float() / (h * w)).view(n, 1, 1, c).expand(n, h, w, c)
        return dx.to(dy.dtype).contiguous()


def maxpool2d(x, kernel=3, stride=2, pad=1):
    return MaxPool2dNHWC.apply(x, kernel, stride, pad)


def global_avgpool(x):
    return GlobalAvgPoolNHWC.apply(x)


# ---------------------------------------------------------------------------
# Linear (MFMA GEMM)
# ---------------------------------------------------------------------------

def _pad_cols64(t):
    """Zero-pad the last dim to a multiple of 64 (GEMM K-dim contract)."""
    k = t.shape[-1]
    r = (-k) % 64
    return t if r == 0 else F.pad(t, (0, r))

class LinearFn(torch.autograd.Function):
    """y = x @ W^T + b; x [M,K] compute dtype, W master fp32 [N,K]."""

    @staticmethod
    def forward(ctx, x, weight, w_packed, bias, w_packed_t=None,
                gslot_w=None, gslot_b=None):
        ctx.save_for_backward(x, weight, w_packed,
                              w_packed_t if w_packed_t is not None
                              else w_packed)
        ctx.has_t = w_packed_t is not None
        ctx.has_bias = bias is not None
        ctx.gslot_w, ctx.gslot_b = gslot_w, gslot_b
        if x.is_cuda:
            return ext().gemm_nt(x, w_packed, bias)
        y = x.float() @ weight.float().t()
        if bias is not None:
            y = y + bias.float()
        return y.to(x.dtype)

    @staticmethod
    def backward(ctx, dy):
        x, weight, w_packed, w_packed_t = ctx.saved_tensors
        dy = dy.contiguous()
        dx = dw = db = None
        if x.is_cuda:
            # every variant is the nt kernel over cheap repacks; K-dims are
            # zero-padded to multiples of 64 (zero rows/cols add nothing)
            if ctx.needs_input_grad[0]:
                dyp = _pad_cols64(dy)
                wtp = _pad_cols64(w_packed_t if ctx.has_t
                                  else w_packed.t().contiguous())
                dx = ext().gemm_nt(dyp, wtp)                  # [M, K_in]
            if ctx.needs_input_grad[1]:
                o_dim, i_dim = weight.shape
                rows = x.shape[0]
                w_out = ctx.gslot_w[0] if ctx.gslot_w is not None else None
                if o_dim % 64 == 0 and i_dim % 64 == 0:
                    # dW = dy^T @ x is exactly the conv-wrw TN GEMM: reuse
                    # its split-K slab kernel (a plain-nt path serialized
                    # K=rows in a handful of blocks — 358us per MLP grad)
                    dw = ext().conv2d_bwd_weight(
                        x.view(1, rows, 1, i_dim), dy.view(1, rows, 1, o_dim),
                        1, 1, 1, 0,
                        out=(w_out.view(o_dim, i_dim, 1, 1)
                             if w_out is not None else None)
                    ).view(o_dim, i_dim)
                else:
                    dyt = _pad_cols64(dy.t().contiguous())    # [O, M]
                    xt = _pad_cols64(x.t().contiguous())      # [K_in, M]
                    dw = ext().gemm_nt(dyt, xt, None, True)   # fp32 [O, K_in]
                    if w_out is not None:
                        w_out.copy_(dw)
                if w_out is not None:
                    if ctx.gslot_w[1] is not None:
                        ctx.gslot_w[1]()
                    dw = None
            if ctx.has_bias and ctx.needs_input_grad[3]:
                db = ext().colsum_f32(
                    dy, out=(ctx.gslot_b[0] if ctx.gslot_b is not None
                             else None))                      # [M,N] -> [N]
                if ctx.gslot_b is not None:
                    if ctx.gslot_b[1] is not None:
                        ctx.gslot_b[1]()
                    db = None
        else:
            dy32, x32, w32 = dy.float(), x.float(), weight.float()
            if ctx.needs_input_grad[0]:
                dx = (dy32 @ w32).to(x.dtype)
            if ctx.needs_input_grad[1]:
                dw = dy32.t() @ x32
            if ctx.has_bias and ctx.needs_input_grad[3]:
                db = dy32.sum(dim=0)
        return dx, dw, None, db, None, None, None


def linear(x, weight, w_packed, bias=None, w_packed_t=None, gslot_w=None,
           gslot_b=None):
    return LinearFn.apply(x, weight, w_packed, bias, w_packed_t, gslot_w,
                          gslot_b)


# ---------------------------------------------------------------------------
# Fused softmax cross-entropy
# ---------------------------------------------------------------------------

class SoftmaxCrossEntropy(torch.autograd.Function):
    """Mean CE over the batch; fused log-softmax + NLL fwd and
    dlogits = (softmax - onehot)/B bwd (SURVEY.md §2d softmax-CE row)."""

    @staticmethod
    def forward(ctx, logits, labels, label_smoothing: float):
        ctx.label_smoothing = label_smoothing
        if logits.is_cuda:
            loss_per, lse = ext().softmax_ce_fwd(logits, labels,
                                                 label_smoothing)
            ctx.save_for_backward(logits, labels, lse)
            return loss_per.mean()
        l32 = logits.float()
        lse = torch.logsumexp(l32, dim=1)
        nll = lse - l32.gather(1, labels.view(-1, 1)).squeeze(1)
        if label_smoothing > 0.0:
            eps = label_smoothing
            smooth = lse - l32.mean(dim=1)
            nll = (1 - eps) * nll + eps * smooth
        ctx.save_for_backward(logits, labels, lse)
        return nll.mean()

    @staticmethod
    def backward(ctx, grad):
        logits, labels, lse = ctx.saved_tensors
        eps = ctx.label_smoothing
        b = logits.shape[0]
        # grad is a device scalar tensor; never .item() it (host sync in the
        # hot loop) — the kernel multiplies by it on device.
        if logits.is_cuda:
            dlogits = ext().softmax_ce_bwd(logits, labels, lse, eps, 1.0 / b,
                                           grad.to(torch.float32))
        else:
            l32 = logits.float()
            p = torch.exp(l32 - lse.unsqueeze(1))
            n = l32.shape[1]
            tgt = F.one_hot(labels, n).float()
            if eps > 0.0:
                tgt = (1 - eps) * tgt + eps / n
            dlogits = ((p - tgt) * (grad.float() / b)).to(logits.dtype)
        return dlogits, None, None


def softmax_cross_entropy(logits, labels, label_smoothing: float = 0.0):
    return SoftmaxCrossEntropy.apply(logits, labels, label_smoothing)


# ---------------------------------------------------------------------------
# Transformer ops (ViT path: LayerNorm, GELU, attention)
# ---------------------------------------------------------------------------

class LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps: float, gslot_w=None,
                gslot_b=None):
        ctx.gslot_w, ctx.gslot_b = gslot_w, gslot_b
        if x.is_cuda:
            y, mean, invstd = ext().ln_fwd(x, weight, bias, eps)
        else:
            x32 = x.float()
            mean = x32.mean(dim=-1)
            var = x32.var(dim=-1, unbiased=False)
            invstd = (var + eps).rsqrt()
            y = ((x32 - mean.unsqueeze(-1)) * invstd.unsqueeze(-1)
                 * weight.float() + bias.float()).to(x.dtype)
        ctx.save_for_backward(x, weight, mean, invstd)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, mean, invstd = ctx.saved_tensors
        dy = dy.contiguous()
        if x.is_cuda:
            dx, dw, db = ext().ln_bwd(
                x, dy, weight, mean, invstd,
                dw_out=ctx.gslot_w[0] if ctx.gslot_w is not None else None,
                db_out=ctx.gslot_b[0] if ctx.gslot_b is not None else None)
            if ctx.gslot_w is not None:
                if ctx.gslot_w[1] is not None:
                    ctx.gslot_w[1]()
                dw = None
            if ctx.gslot_b is not None:
                if ctx.gslot_b[1] is not None:
                    ctx.gslot_b[1]()
                db = None
        else:
            d = x.shape[-1]
            x32, g32, w32 = x.float(), dy.float(), weight.float()
            xhat = (x32 - mean.unsqueeze(-1)) * invstd.unsqueeze(-1)
            gw = g32 * w32
            s1 = gw.mean(dim=-1, keepdim=True)
            s2 = (gw * xhat).mean(dim=-1, keepdim=True)
            dx = (invstd.unsqueeze(-1) * (gw - s1 - xhat * s2)).to(x.dtype)
            dims = tuple(range(x.dim() - 1))
            dw = (g32 * xhat).sum(dim=dims)
            db = g32.sum(dim=dims)
        return dx, dw, db, None, None, None


def layer_norm(x, weight, bias, eps: float = 1e-6, gslot_w=None,
               gslot_b=None):
    return LayerNormFn.apply(x, weight, bias, eps, gslot_w, gslot_b)



class AddLayerNormFn(torch.autograd.Function):
    """Fused residual join + LayerNorm: (y, s) = (ln(a+b), a+b).

    The ViT block threads (residual, branch) PAIRS between sublayers so
    the sum has exactly ONE consumer — no autograd fork add exists in
    either direction. Backward folds the pass-through gradient ds into
    the dx store (DXADD kernel variant) and returns the SAME combined
    gradient for both inputs."""

    @staticmethod
    def forward(ctx, a, b, weight, bias, eps, gslot_w=None, gslot_b=None):
        ctx.set_materialize_grads(False)
        ctx.gslot_w, ctx.gslot_b = gslot_w, gslot_b
        if a.is_cuda:
            y, mean, invstd, s = ext().ln_fwd(a, weight, bias, eps,
                                              res=b.contiguous())
        else:
            s = (a.float() + b.float()).to(a.dtype)
            s32 = s.float()
            mean = s32.mean(dim=-1)
            var = s32.var(dim=-1, unbiased=False)
            invstd = (var + eps).rsqrt()
            y = ((s32 - mean.unsqueeze(-1)) * invstd.unsqueeze(-1)
                 * weight.float() + bias.float()).to(a.dtype)
        ctx.save_for_backward(s, weight, mean, invstd)
        return y, s

    @staticmethod
    def backward(ctx, dy, ds):
        s, weight, mean, invstd = ctx.saved_tensors
        dy = dy.contiguous()
        if s.is_cuda:
            dx, dw, db = ext().ln_bwd(
                s, dy, weight, mean, invstd,
                dxadd=ds.contiguous() if ds is not None else None,
                dw_out=ctx.gslot_w[0] if ctx.gslot_w is not None else None,
                db_out=ctx.gslot_b[0] if ctx.gslot_b is not None else None)
            if ctx.gslot_w is not None:
                if ctx.gslot_w[1] is not None:
                    ctx.gslot_w[1]()
                dw = None
            if ctx.gslot_b is not None:
                if ctx.gslot_b[1] is not None:
                    ctx.gslot_b[1]()
                db = None
        else:
            d = s.shape[-1]
            s32, g32, w32 = s.float(), dy.float(), weight.float()
            xhat = (s32 - mean.unsqueeze(-1)) * invstd.unsqueeze(-1)
            gw = g32 * w32
            s1 = gw.mean(dim=-1, keepdim=True)
            s2 = (gw * xhat).mean(dim=-1, keepdim=True)
            dx = (invstd.unsqueeze(-1) * (gw - s1 - xhat * s2))
            if ds is not None:
                dx = dx + ds.float()
            dx = dx.to(s.dtype)
            dims = tuple(range(s.dim() - 1))
            dw = (g32 * xhat).sum(dim=dims)
            db = g32.sum(dim=dims)
        return dx, dx, dw, db, None, None, None


def add_layer_norm(a, b, weight, bias, eps: float = 1e-6, gslot_w=None,
                   gslot_b=None):
    return AddLayerNormFn.apply(a, b, weight, bias, eps, gslot_w, gslot_b)


class GELUFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        ctx.save_for_backward(x)
        if x.is_cuda:
            return ext().gelu_fwd(x)
        return F.gelu(x.float()).to(x.dtype)

    @staticmethod
    def backward(ctx, dy):
        (x,) = ctx.saved_tensors
        dy = dy.contiguous()
        if x.is_cuda:
            return ext().gelu_bwd(x, dy)
        x32 = x.float().detach().requires_grad_()
        with torch.enable_grad():
            y = F.gelu(x32)
        (dx,) = torch.autograd.grad(y, x32, dy.float())
        return dx.to(x.dtype)


def gelu(x):
    return GELUFn.apply(x)


class AttentionFn(torch.autograd.Function):
    """Scaled-dot-product attention over padded sequences.

    q,k,v: [bat, S, hd] (S padded to a multiple of 64; hd % 64 == 0);
    columns >= nvalid are masked out of the softmax, padded v rows are
    zero, so results for rows < nvalid are exact. GPU path: batched MFMA
    GEMMs (QK^T fp32) + fused masked-softmax kernel (SURVEY.md §2d ViT
    attention row).
    """

    @staticmethod
    def forward(ctx, q, k, v, nvalid: int, scale: float):
        if q.is_cuda:
            scores = ext().gemm_nt_batched(q, k, True)        # fp32 [b,S,S]
            p = ext().attn_softmax_fwd(scores, nvalid, scale, q.dtype)
            vt = v.transpose(1, 2).contiguous()               # [b, hd, S]
            out = ext().gemm_nt_batched(p, vt)                # [b, S, hd]
        else:
            s32 = (q.float() @ k.float().transpose(1, 2)) * scale
            mask = torch.arange(q.shape[1]) >= nvalid
            s32 = s32.masked_fill(mask.view(1, 1, -1), float("-inf"))
            p32 = torch.softmax(s32, dim=-1)
            p = p32.to(q.dtype)
            out = (p32 @ v.float()).to(q.dtype)
        ctx.save_for_backward(q, k, v, p)
        ctx.scale = scale
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, p = ctx.saved_tensors
        dout = dout.contiguous()
        scale = ctx.scale
        if q.is_cuda:
            dp = ext().gemm_nt_batched(dout, v)               # [b, S, S]
            ds = ext().attn_softmax_bwd(p, dp, scale).to(q.dtype)
            kt = k.transpose(1, 2).contiguous()               # [b, hd, S]
            dq = ext().gemm_nt_batched(ds, kt)                # [b, S, hd]
            dst = ds.transpose(1, 2).contiguous()
            qt = q.transpose(1, 2).contiguous()
            dk = ext().gemm_nt_batched(dst, qt)
            pt = p.transpose(1, 2).contiguous()
            dot = dout.transpose(1, 2).contiguous()
            dv = ext().gemm_nt_batched(pt, dot)
        else:
            p32, g32 = p.float(), dout.float()
            dp = g32 @ v.float().transpose(1, 2)
            ds = (p32 * (dp - (p32 * dp).sum(-1, keepdim=True)) * scale)
            dq = (ds @ k.float()).to(q.dtype)
            dk = (ds.transpose(1, 2) @ q.float()).to(q.dtype)
            dv = (p32.transpose(1, 2) @ g32).to(q.dtype)
        return dq, dk, dv, None, None


def attention(q, k, v, nvalid: int, scale: float):
    return AttentionFn.apply(q, k, v, nvalid, scale)


class AttentionQKVFn(torch.autograd.Function):
    """Zero-copy multi-head attention over the interleaved qkv projection
    [b*s, 3*h*hd]: q/k/v are consumed IN PLACE via strided-batched MFMA
    GEMMs and all gradients are written IN PLACE into d(qkv) — no
    permute/contiguous copies anywhere (those were 30% of the ViT step).
    GPU-only; the CPU path uses AttentionFn via explicit permutes.
    """

    @staticmethod
    def forward(ctx, qkv2d, b: int, s: int, h: int, hd: int, nvalid: int,
                scale: float):
        qkv3 = qkv2d.view(b, s, 3 * h * hd)
        out, p = ext().attn_fwd(qkv3, b, s, h, hd, nvalid, scale)
        ctx.save_for_backward(qkv2d, p)
        ctx.dims = (b, s, h, hd, nvalid, scale)
        return out  # [b, s, h*hd]

    @staticmethod
    def backward(ctx, dout):
        qkv2d, p = ctx.saved_tensors
        b, s, h, hd, nvalid, scale = ctx.dims
        dqkv = ext().attn_bwd(qkv2d.view(b, s, 3 * h * hd), p,
                              dout.contiguous(), b, s, h, hd, nvalid,
                              scale)
        return dqkv.view(b * s, 3 * h * hd), None, None, None, None, None, \
            None


def attention_qkv(qkv2d, b, s, h, hd, nvalid, scale):
    return AttentionQKVFn.apply(qkv2d, b, s, h, hd, nvalid, scale)


# ---------------------------------------------------------------------------
# Attention with recomputed probabilities
# ---------------------------------------------------------------------------

def _visible(q, k, causal, q_lens, kv_lens):
    """[b, 1, 1, sq, sk] where a query may see a key, for the CPU path."""
    sq, sk = q.shape[1], k.shape[1]
    i, j = torch.arange(sq)[:, None], torch.arange(sk)[None, :]
    at = (-1, 1, 1, 1, 1)
    ql = torch.tensor([sq]) if q_lens is None else q_lens.long().clamp(0, sq)
    kl = torch.tensor([sk]) if kv_lens is None \
        else kv_lens.long().clamp(0, sk)
    ql, kl = ql.view(at), kl.view(at)
    ok = (i < ql) & (j < kl)
    if causal:
        ok = ok & (j <= i + kl - ql)
    return ok


class AttentionRecomputeFn(torch.autograd.Function):
    """CPU reference; the GPU path's node is C++ (bind_transformer.cpp)."""

    @staticmethod
    def forward(ctx, q, k, v, scale, causal, q_lens, kv_lens):
        ctx.scale, ctx.causal = scale, causal
        b, sq, h, hd = q.shape
        hk = k.shape[2]
        ok = _visible(q, k, causal, q_lens, kv_lens)
        # what is masked may hold anything: 0 * inf must not come up
        seen_k = ok.any(3)[:, 0, 0, :, None, None]
        seen_q = ok.any(4)[:, 0, 0, :, None, None]
        q5, k5, v5 = (_heads_first(_wide(x).masked_fill(~m, 0.0), hk)
                      for x, m in ((q, seen_q), (k, seen_k), (v, seen_k)))
        s = (q5 @ k5.transpose(-1, -2)) * scale
        lse = s.masked_fill(~ok, float("-inf")).logsumexp(-1, keepdim=True)
        lse = lse.masked_fill(lse == float("-inf"), float("inf"))
        p = (s - lse).exp().masked_fill(~ok, 0.0)
        out = _heads_last(p @ v5, h).to(q.dtype)
        ctx.save_for_backward(q, k, v, out, lse, q_lens, kv_lens)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, q_lens, kv_lens = ctx.saved_tensors
        scale, causal = ctx.scale, ctx.causal
        h, hk = q.shape[2], k.shape[2]
        ok = _visible(q, k, causal, q_lens, kv_lens)
        seen_k = ok.any(3)[:, 0, 0, :, None, None]
        seen_q = ok.any(4)[:, 0, 0, :, None, None]
        q5, k5, v5, o5, g5 = (
            _heads_first(_wide(x).masked_fill(~m, 0.0), hk)
            for x, m in ((q, seen_q), (k, seen_k), (v, seen_k),
                         (out, seen_q), (dout, seen_q)))
        p = ((q5 @ k5.transpose(-1, -2)) * scale - lse).exp() \
            .masked_fill(~ok, 0.0)
        dv = (p.transpose(-1, -2) @ g5).sum(2, keepdim=True)
        ds = p * (g5 @ v5.transpose(-1, -2)
                  - (g5 * o5).sum(-1, keepdim=True)) * scale
        dq = _heads_last(ds @ k5, h).to(q.dtype)
        dk = (ds.transpose(-1, -2) @ q5).sum(2, keepdim=True)
        return (dq, _heads_last(dk, hk).to(k.dtype),
                _heads_last(dv, hk).to(v.dtype), None, None, None, None)


def _heads_first(x, hk):
    # [b, s, h, hd] -> [b, hk, h/hk, s, hd]
    b, s, h, hd = x.shape
    return x.view(b, s, hk, h // hk, hd).permute(0, 2, 3, 1, 4)


def _heads_last(x, h):
    b, _, _, s, hd = x.shape
    return x.permute(0, 3, 1, 2, 4).reshape(b, s, h, hd).contiguous()


def attention_recompute(q, k, v, scale: float | None = None,
                        causal: bool = False, q_lens=None, kv_lens=None):
    """softmax(scale q k^T) v without an sq x sk tensor in either direction:
    the forward keeps each row's log-sum-exp, the backward recomputes the
    probabilities from it. Returns [b, sq, h, hd], contiguous.

    q [b, sq, h, hd], k, v [b, sk, hk, hd]; h a multiple of hk: h/hk
    neighbouring query heads share a key head. Any strides (the views of one
    projection's output need no copy when their rows are 16-byte aligned).
    scale: positive, None for 1/sqrt(hd).
    q_lens, kv_lens: int32 or int64 [b], the sequences' lengths (None: sq,
    sk); cut to 0..sq, 0..sk. What lies behind them is never read; outputs
    and gradients there are 0. Inside them every element has to be finite: a
    pair that the causal mask hides counts 0 times what it holds, which does
    not keep a NaN or an infinity from the other rows of its tile.
    causal: query i sees keys up to i + kv_len - q_len, so the last query
    sees the last key. A query that sees none gives 0.
    GPU (csrc/attn_recompute.hip): bf16 and fp16, hd a multiple of 8 up to
    128; results do not depend on timing; no gradient of the gradient. A
    captured forward that needs gradients is refused while another graph of
    the same leaves, made on the default stream, is alive.
    In fp16, gradients need a loss scale that keeps dS in its range, as the
    fp16 training path has."""
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape \
            or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError("q must be [b, sq, h, hd], k and v [b, sk, hk, hd]: "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    b, h, hk, hd = q.shape[0], q.shape[2], k.shape[2], q.shape[3]
    if hk == 0 or h % hk or hd == 0:
        raise ValueError(f"{h} query heads for {hk} key heads of {hd}")
    if not q.dtype == k.dtype == v.dtype \
            or not q.device == k.device == v.device:
        raise ValueError("q, k and v must have one dtype and device")
    if q.is_cuda and (hd % 8 or hd > 128):
        raise ValueError(f"head size must be a multiple of 8 up to 128: {hd}")
    if scale is None:
        scale = hd ** -0.5
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"scale must be positive: {scale}")
    for x in (q_lens, kv_lens):
        if x is not None and (x.shape != (b,) or x.device != q.device
                              or x.dtype not in (torch.int32, torch.int64)):
            raise ValueError(f"lengths must be int32 or int64 [{b}] on "
                             f"{q.device}")
    if q_lens is not None and kv_lens is not None \
            and q_lens.dtype != kv_lens.dtype:
        q_lens, kv_lens = q_lens.long(), kv_lens.long()
    q_lens, kv_lens = (x if x is None else x.contiguous()
                       for x in (q_lens, kv_lens))
    if q.is_cuda:
        return ext().attention_recompute(q, k, v, q_lens, kv_lens, scale,
                                         causal)
    return AttentionRecomputeFn.apply(q, k, v, float(scale), bool(causal),
                                      q_lens, kv_lens)


# ---------------------------------------------------------------------------
# Query/key norm with the position rotation
# ---------------------------------------------------------------------------

def rope_tables(n: int, rot_dim: int, theta: float = 10000.0,
                scale: float = 1.0, device=None):
    """(cos, sin), fp32 [n, rot_dim/2], of the angles
    position / scale * theta^(-2i/rot_dim). scale > 1 squeezes longer
    sequences into the positions a model has seen. Angles are formed in 64
    bits: in 32 those of far positions are off by more than 1e-3."""
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rot_dim must be even and positive: {rot_dim}")
    f = theta ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64,
                                device=device) / rot_dim)
    a = torch.arange(n, dtype=torch.float64, device=device) / scale
    a = a[:, None] * f
    return a.cos().float(), a.sin().float()


def rope_tables_2d(rows: int, cols: int, rot_dim: int, theta: float = 100.0,
                   prefix: int = 0, device=None):
    """(cos, sin), fp32 [prefix + rows*cols, rot_dim/2], for a grid of
    patches in row order: half of the angles turn with the row, half with
    the column. `prefix` tokens before the grid (a class token) do not
    turn."""
    if rot_dim % 4:
        raise ValueError(f"rot_dim must be a multiple of 4: {rot_dim}")
    r, c = (rope_tables(n, rot_dim // 2, theta, device=device)
            for n in (rows, cols))
    out = []
    for x, y, still in zip(r, c, (1.0, 0.0)):
        grid = torch.cat([x[:, None].expand(rows, cols, -1),
                          y[None].expand(rows, cols, -1)], -1)
        out.append(torch.cat([x.new_full((prefix, rot_dim // 2), still),
                              grid.reshape(rows * cols, -1)]))
    return tuple(out)


def _wide(x):
    # the CPU reference computes in fp32; fp64 stays, for differences
    return x if x.dtype == torch.float64 else x.float()


def _rotate(x, cos, sin, interleaved):
    """x [b, s, h, hd] with its first 2*cos.shape[-1] elements turned;
    cos, sin [b or 1, s, 1, rot/2]."""
    half = cos.shape[-1]
    rot = 2 * half
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:rot]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _gathered(cos, sin, positions, s):
    """Rows of the tables for every token; a position outside them turns by
    NaN, as in the kernel."""
    if positions is None:
        return cos[:s][None, :, None], sin[:s][None, :, None]
    ok = (positions >= 0) & (positions < cos.shape[0])
    at = positions.long().clamp(0, cos.shape[0] - 1)
    bad = (~ok)[:, :, None]
    return tuple(t[at].masked_fill(bad, float("nan"))[:, :, None]
                 for t in (cos, sin))


class QKNormRopeFn(torch.autograd.Function):
    """CPU reference; the GPU path's node is C++ (bind_transformer.cpp)."""

    @staticmethod
    def forward(ctx, q, k, wq, wk, cos, sin, positions, eps, interleaved):
        ctx.eps, ctx.interleaved = eps, interleaved
        ctx.save_for_backward(q, k, wq, wk, cos, sin, positions)

        def one(x, w):
            x32 = _wide(x)
            if w is not None:
                r = (x32.square().mean(-1, keepdim=True) + eps).rsqrt()
                x32 = x32 * r * _wide(w)
            if cos is not None:
                c, s = _gathered(cos, sin, positions, x.shape[1])
                x32 = _rotate(x32, c, s, interleaved)
            return x32.to(x.dtype)

        return one(q, wq), one(k, wk)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        q, k, wq, wk, cos, sin, positions = ctx.saved_tensors

        def one(x, w, dy):
            g = _wide(dy)
            if cos is not None:
                c, s = _gathered(cos, sin, positions, x.shape[1])
                g = _rotate(g, c, -s, ctx.interleaved)
            if w is None:
                return g.to(x.dtype), None
            x32 = _wide(x)
            r = (x32.square().mean(-1, keepdim=True) + ctx.eps).rsqrt()
            xhat = x32 * r
            dw = (g * xhat).sum((0, 1, 2))
            g = g * _wide(w)
            dx = r * (g - xhat * (g * xhat).mean(-1, keepdim=True))
            return dx.to(x.dtype), dw

        dq, dwq = one(q, wq, dq)
        dk, dwk = one(k, wk, dk)
        return dq, dk, dwq, dwk, None, None, None, None, None


def qk_norm_rope(q, k, q_weight=None, k_weight=None, cos=None, sin=None,
                 positions=None, eps: float = 1e-6,
                 interleaved: bool = False):
    """RMS norm of every query and key head with the position rotation in
    the same pass: (q', k'), contiguous.

    q [b, s, h, hd], k [b, s, hk, hd]: bf16, fp16 or fp32, any strides (the
    views of one projection's output need no copy), hd up to 256.
    q_weight, k_weight: fp32 [hd], both or neither (no norm).
    cos, sin: fp32 [positions, rot/2] (rope_tables), both or neither (no
    rotation); rot <= hd, the rest of the head is left as it is. Pairs are
    (i, i + rot/2), or (2i, 2i+1) when interleaved.
    positions: int32 or int64 [b, s], None for 0..s-1. One outside the
    tables turns by NaN. The tables have no gradient.
    GPU: csrc/qknorm.hip, one launch (two in backward); 16-byte accesses
    where hd % 8 == 0, rot % 16 == 0 (8 interleaved) and rows are aligned."""
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] \
            or q.shape[3] != k.shape[3]:
        raise ValueError("q and k must be [b, s, heads, hd], alike but for "
                         f"the heads: {tuple(q.shape)}, {tuple(k.shape)}")
    if q.dtype != k.dtype or q.device != k.device:
        raise ValueError("q and k must have one dtype and device")
    b, s, hd = q.shape[0], q.shape[1], q.shape[3]
    if not 1 <= hd <= 256:
        raise ValueError(f"head size must be 1 to 256: {hd}")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("q_weight and k_weight come together")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if q_weight is None and cos is None:
        raise ValueError("neither weights nor tables: nothing to do")
    for w in (q_weight, k_weight):
        if w is not None and w.shape != (hd,):
            raise ValueError(f"weights must be [{hd}]: {tuple(w.shape)}")
    if cos is not None:
        if cos.dim() != 2 or cos.shape != sin.shape \
                or not 2 <= 2 * cos.shape[1] <= hd:
            raise ValueError("cos and sin must be [positions, rot/2] with "
                             f"rot <= {hd}: {tuple(cos.shape)}, "
                             f"{tuple(sin.shape)}")
        if cos.requires_grad or sin.requires_grad:
            raise ValueError("cos and sin have no gradient")
        if positions is None and s > cos.shape[0]:
            raise ValueError(f"tables for {cos.shape[0]} positions, "
                             f"sequences of {s}")
    if positions is not None and (
            positions.shape != (b, s)
            or positions.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"positions must be int32 or int64 [{b}, {s}]")
    positions, cos, sin, q_weight, k_weight = (
        x if x is None else x.contiguous()
        for x in (positions, cos, sin, q_weight, k_weight))
    if q.is_cuda:
        return tuple(ext().qk_norm_rope_grad(q, k, q_weight, k_weight, cos,
                                             sin, positions, eps,
                                             interleaved))
    return QKNormRopeFn.apply(q, k, q_weight, k_weight, cos, sin, positions,
                              eps, interleaved)


class AttentionQKVRopeFn(torch.autograd.Function):
    """qk_norm_rope and attention_recompute over one projection's output
    [b*s, 3*h*hd], as attention_qkv: q, k and v are read in place, and
    backward writes its three parts of d(qkv) in place, so nothing is split,
    stacked or copied. GPU only; the CPU path composes the two."""

    @staticmethod
    def forward(ctx, qkv2d, wq, wk, cos, sin, b, s, h, hd, scale, causal,
                eps, gslot_q, gslot_k):
        q, k, v = qkv2d.view(b, s, 3, h, hd).unbind(2)
        qn, kn = ext().qk_norm_rope(q, k, wq, wk, cos, sin, None, eps, False)
        out, lse = ext().attn_recompute_fwd(qn, kn, v, None, None, scale,
                                            causal, True)
        ctx.save_for_backward(qkv2d, wq, wk, cos, sin, qn, kn, out, lse)
        ctx.dims = (b, s, h, hd, scale, causal, eps)
        ctx.gslot = (gslot_q, gslot_k)
        return out.view(b, s, h * hd)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        qkv2d, wq, wk, cos, sin, qn, kn, out, lse = ctx.saved_tensors
        b, s, h, hd, scale, causal, eps = ctx.dims
        q, k, v = qkv2d.view(b, s, 3, h, hd).unbind(2)
        dqkv = torch.empty_like(qkv2d)
        dq, dk, dv = dqkv.view(b, s, 3, h, hd).unbind(2)
        dqn, dkn, _ = ext().attn_recompute_bwd(
            qn, kn, v, out, lse, dout.contiguous().view(b, s, h, hd), None,
            None, scale, causal, dv_out=dv)
        dw = [torch.empty_like(w) if slot is None else slot[0]
              for w, slot in zip((wq, wk), ctx.gslot)]
        ext().qk_norm_rope(q, k, wq, wk, cos, sin, None, eps, False, dq=dqn,
                           dk=dkn, outs=[dq, dk, *dw])
        for i, slot in enumerate(ctx.gslot):
            if slot is not None:
                dw[i] = None
                if slot[1] is not None:
                    slot[1]()
        return (dqkv, *dw) + (None,) * 11


def attention_qkv_rope(qkv2d, q_weight, k_weight, cos, sin, b: int, s: int,
                       h: int, hd: int, scale: float | None = None,
                       causal: bool = False, eps: float = 1e-6,
                       gslot_q=None, gslot_k=None):
    """Multi-head attention over the interleaved projection [b*s, 3*h*hd]
    with normed and rotated queries and keys (qk_norm_rope, halves layout)
    and no s x s tensor (attention_recompute): [b, s, h*hd]. Gradients of
    the projection come in its layout; of the weights directly into gslot_q,
    gslot_k when given."""
    if qkv2d.shape != (b * s, 3 * h * hd):
        raise ValueError(f"qkv must be [{b * s}, {3 * h * hd}]: "
                         f"{tuple(qkv2d.shape)}")
    if q_weight is None or k_weight is None:
        raise ValueError("q_weight and k_weight must be given")
    if any(t is not None and t.requires_grad for t in (cos, sin)):
        raise ValueError("cos and sin have no gradient")
    if scale is None:
        scale = hd ** -0.5
    if qkv2d.is_cuda:
        ext().capture_check([qkv2d, q_weight, k_weight])
        return AttentionQKVRopeFn.apply(qkv2d.contiguous(), q_weight,
                                        k_weight, cos, sin, b, s, h, hd,
                                        scale, causal, eps, gslot_q, gslot_k)
    q, k, v = qkv2d.view(b, s, 3, h, hd).unbind(2)
    q, k = qk_norm_rope(q, k, q_weight, k_weight, cos, sin, eps=eps)
    return attention_recompute(q, k, v, scale=scale, causal=causal) \
        .view(b, s, h * hd)


# ---------------------------------------------------------------------------
# AdamW over flat storage
# ---------------------------------------------------------------------------

ADAMW_BLOCK = 64          # elements under one 8-bit scale, one decay byte
_ADAMW_TINY = 2.0 ** -100  # a block whose largest is below is stored as 0


def _scale8(x):
    top = x.abs().view(-1, ADAMW_BLOCK).amax(1)
    dead = top < _ADAMW_TINY
    scale = (top * (1.0 / 448.0)).masked_fill(dead, 0.0)
    inv = (top.reciprocal() * 448.0).masked_fill(dead, 0.0)
    return scale, inv.repeat_interleave(ADAMW_BLOCK)


def adamw_quantize(x, positive: bool = False):
    """fp32 [n] -> (float8_e4m3fn [n], fp32 scale [n/64]), to the nearest;
    x is about value * scale of its block of 64. positive (x >= 0): what is
    above 0 stays above 0, as sqrt(v) has to."""
    scale, inv = _scale8(x)
    y = (x * inv).clamp(-448.0, 448.0)
    if positive:
        y = torch.where(y > 0, y.clamp(min=2.0 ** -9), y)
    return y.to(torch.float8_e4m3fn), scale


def adamw_dequantize(codes, scale):
    """Inverse of adamw_quantize, in fp32."""
    return codes.float() * scale.repeat_interleave(ADAMW_BLOCK)


def _adamw_noise(n, step, seed, device):
    # 16 random bits an element: the halves of a mix of its pair's index,
    # the step and the seed, as in csrc/adamw.hip
    low = 0xFFFFFFFF
    x = torch.arange(n // 2, dtype=torch.int64, device=device)
    x = (x * 0x9E3779B1 + step * 0x6A09E667 + seed * 0x3B67AE85) & low
    x = ((x ^ (x >> 16)) * 0x3C6EF373) & low
    x = ((x ^ (x >> 15)) * 0x254FF53B) & low
    x = x ^ (x >> 16)
    return torch.stack([x & 0xFFFF, x >> 16], 1).view(-1).float()


def _adamw_quantize_random(x, step, seed):
    scale, inv = _scale8(x)
    y = (x * inv).clamp(max=448.0)
    # the distance of neighbouring e4m3 values: 2^(exponent - 3)
    unit = torch.ldexp(torch.ones_like(y),
                       torch.frexp(y.clamp(min=2.0 ** -6))[1] - 4)
    r = _adamw_noise(x.numel(), step, seed, x.device) * 2.0 ** -16
    z = (torch.floor(y / unit + r) * unit).clamp(max=448.0)
    z = torch.where(y > 0, z.clamp(min=2.0 ** -9), y)
    return z.to(torch.float8_e4m3fn), scale


@torch.no_grad()
def adamw_step(p, g, m, v, step, lr, beta1=0.9, beta2=0.999, eps=1e-8,
               weight_decay=0.01, decay=None, grad_scale=1.0, m_scale=None,
               v_scale=None, seed=0):
    """One AdamW step in place over flat fp32 storage p with gradient g
    (torch.optim.AdamW's formula; n a multiple of 64):

        step += 1;  g = g * grad_scale
        m = beta1 m + (1-beta1) g;   v = beta2 v + (1-beta2) g^2
        p = p (1 - lr weight_decay decay)
              - lr/(1-beta1^step) m / (sqrt(v)/sqrt(1-beta2^step) + eps)

    step: one int64 on p's device, advanced here, so a captured step replays
    as the next one. lr: a number, or one float32 on p's device.
    decay: None, or uint8 [n/64], 1 where weight decay applies, 0 elsewhere.
    States: m, v fp32; or, with m_scale and v_scale (fp32 [n/64]),
    float8_e4m3fn of m and of sqrt(v) over a scale per 64 elements, sqrt(v)
    rounded up or down at random by a mix of element, step and seed. A
    gradient that is not finite makes p's element NaN and its block's 8-bit
    state not finite. GPU: csrc/adamw.hip, two launches."""
    if not (0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0):
        raise ValueError(f"betas must be in [0, 1): {beta1}, {beta2}")
    if eps < 0.0:
        raise ValueError(f"eps must not be negative: {eps}")
    n = p.numel()
    if n % ADAMW_BLOCK:
        raise ValueError(f"p must have a multiple of {ADAMW_BLOCK} elements, "
                         f"has {n}")
    if (m_scale is None) != (v_scale is None):
        raise ValueError("m_scale and v_scale come together")
    lr_dev = lr if isinstance(lr, torch.Tensor) else None
    if p.is_cuda:
        ext().adamw_step(p, g, m, v, step,
                         0.0 if lr_dev is not None else float(lr), lr_dev,
                         beta1, beta2, eps, weight_decay, decay, grad_scale,
                         m_scale, v_scale, seed & 0xFFFFFFFF)
        return
    state = torch.float32 if m_scale is None else torch.float8_e4m3fn
    for name, t, dtype, size in (
            ("p", p, torch.float32, n), ("g", g, torch.float32, n),
            ("m", m, state, n), ("v", v, state, n),
            ("m_scale", m_scale, torch.float32, n // ADAMW_BLOCK),
            ("v_scale", v_scale, torch.float32, n // ADAMW_BLOCK),
            ("decay", decay, torch.uint8, n // ADAMW_BLOCK),
            ("step", step, torch.int64, 1)):
        if t is not None and (t.dtype != dtype or t.numel() != size
                              or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous {dtype} with "
                             f"{size} elements")
    step += 1
    t = int(step)
    if lr_dev is not None:
        lr = float(lr_dev)
    if m_scale is None:
        m32, v32 = m, v
    else:
        m32 = adamw_dequantize(m, m_scale)
        v32 = adamw_dequantize(v, v_scale).square_()
    gs = g if grad_scale == 1.0 else g * grad_scale
    m32.mul_(beta1).add_(gs * (1.0 - beta1))
    v32.mul_(beta2).add_(gs * gs * (1.0 - beta2))
    on = 1.0 if decay is None \
        else decay.repeat_interleave(ADAMW_BLOCK).float()
    p.mul_(1.0 - lr * weight_decay * on)
    bc1, bc2 = 1.0 - beta1 ** t, 1.0 - beta2 ** t
    p.sub_((lr / bc1) * m32 / (v32.sqrt() / bc2 ** 0.5 + eps))
    if m_scale is not None:
        for (codes, scale), (c, s) in (
                (adamw_quantize(m32), (m, m_scale)),
                (_adamw_quantize_random(v32.sqrt(), t, seed & 0xFFFFFFFF),
                 (v, v_scale))):
            c.copy_(codes)
            s.copy_(scale)
