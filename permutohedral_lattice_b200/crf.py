"""Mean-field inference of a dense CRF around the lattice filter: the caller the reference library was
written for (README.md:15-16 of MiguelMonteiro/permutohedral_lattice names CRF-as-RNN; the library itself
ships no CRF code, so this module follows the published mean-field update, not a reference file).

One iteration, for label distributions Q[B, *S, L], unaries U[B, *S, L] (negative log-likelihoods) and a
guide image I[B, *S, R]:

    Qb = lattice_filter(Q, I, bilateral=True,  theta_alpha, theta_beta)      appearance kernel
    Qs = lattice_filter(Q, I, bilateral=False, theta_gamma)                  smoothness kernel
    message  = bilateral_weight * Qb + spatial_weight * Qs
    pairwise = message @ compatibility                                       [L, L], Potts by default
    Q        = softmax(-U - pairwise)

Both lattices depend on the image only: they are built once (`Lattice`) and applied in every iteration.
Everything after the two filters (weights, compatibility product, unaries, softmax) is one fused kernel,
pl_crf_update_f32: one read of Qb, Qs and U and one write of Q per iteration.  For the Potts model on RGB images with 4 to 31
labels the whole iteration is pl_crf_step_f32: each stage of both filters in one launch, the update in the slice.

Training (CRF-as-RNN): `infer` and `step` are differentiable in the unaries, and in the parameters that are given as
tensors: the kernels' weights (one each, or one a label), the compatibility and a bias of the labels.  A step with learned
parameters is

    Q = softmax(label_bias - U - (bilateral_weight * Qb + spatial_weight * Qs) @ compatibility)

as two filters and one `channel_mix`, whose backward pass gives every gradient in one pass over the points; the filters'
gradients are the lattices' applied in reverse.  checkpoint="8bit" keeps a step's distributions in 8 bits until then.

A label is forbidden by an infinite unary; a point without any (padding) has zeros from the start on, sends nothing and takes
no gradient.
"""
import torch
from torch.autograd.function import once_differentiable

from . import capi
from .channel_mix import MixSaved, PackedActivations, channel_mix, channel_mix_backward, pack_activations
from .channel_mix import _backward as _mix_backward
from .lattice_filter import Lattice, _OnDevice, _check_tensor, _float32_only, _stream_handle, _watched_by_torch


class _LatticeApplyFunction(torch.autograd.Function):
    """A kept lattice as a layer: its gradient is the same lattice applied in reverse (lattice_filter_op_loader.py:32-54)."""

    @staticmethod
    def forward(ctx, lattice, x):
        ctx.lattice = lattice
        return lattice.apply(x)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return None, ctx.lattice.apply(grad, reverse=True)


def _start_kernel(unaries):
    u = unaries.contiguous()
    q = torch.empty_like(u)
    with _OnDevice(u.device):
        capi.check(capi.lib().pl_crf_start_f32(q.data_ptr(), u.data_ptr(), u.numel() // u.shape[-1], u.shape[-1],
                                               _stream_handle(u.device)), "pl_crf_start_f32")
    return q


class _CrfStartFunction(torch.autograd.Function):
    """softmax(-unaries) by the kernel that inference starts with.  Its gradient is a step's, without messages."""

    @staticmethod
    def forward(ctx, unaries):
        out = _start_kernel(unaries)
        ctx.save_for_backward(out)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (out,) = ctx.saved_tensors
        weight = out.new_empty((1, out.shape[-1]))       # of no input: this gradient does not depend on it
        return _mix_backward(out.device, grad, out, None, None, weight, None, "softmax", -1.0, ("residual",)).residual


class _CrfStepFunction(torch.autograd.Function):
    """A step with constant parameters, by the kernels that inference takes.  Its gradient needs nothing but its output."""

    @staticmethod
    def forward(ctx, crf, q, unaries):
        out = crf._constant_step(q, unaries)
        ctx.crf, ctx.weights = crf, (crf.bilateral_weight, crf.spatial_weight)
        ctx.packed = None
        compatibility = None if crf.compatibility is None else crf._as_taken(crf.compatibility, out.device)
        if crf.checkpoint:
            packed = pack_activations(out)
            ctx.packed = packed.shape, packed.dtype
            ctx.save_for_backward(compatibility, packed.codes, packed.scales)
        else:
            ctx.save_for_backward(compatibility, out)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        compatibility, *kept = ctx.saved_tensors
        out = kept[0] if ctx.packed is None else PackedActivations(*kept, *ctx.packed)
        crf = ctx.crf
        if compatibility is None:
            compatibility = crf._potts(grad.device)
        wb, ws = (-w * compatibility for w in ctx.weights)
        needs = (("x", "x2") if ctx.needs_input_grad[1] else ()) + (("residual",) if ctx.needs_input_grad[2] else ())
        d = channel_mix_backward(grad, MixSaved(None, None, out), wb, ws, "softmax", -1.0, needs)
        dq = None
        if ctx.needs_input_grad[1]:
            dq = crf.bilateral.apply(d.x, reverse=True)
            dq += crf.spatial.apply(d.x2, reverse=True)
        return None, dq, d.residual


class DenseCRF:
    def __init__(self, image, n_labels, theta_alpha=80.0, theta_beta=0.0625, theta_gamma=3.0,
                 bilateral_weight=1.0, spatial_weight=1.0, compatibility=None, label_bias=None, checkpoint=None):
        """image [B, *S, R] float32 on the GPU; compatibility [L, L] (default: Potts, 1 - identity).
        bilateral_weight, spatial_weight: numbers, or tensors of one value or [L] (a weight for each label that sends
        messages); label_bias: None or [L].  Tensors that require grad are learned: every step takes them as they are then,
        whatever their device, type or order; other tensors are constants, taken now.  checkpoint: None or "8bit", how the steps
        keep what their backward pass needs."""
        shape = tuple(image.shape[:-1])
        self.n_labels = int(n_labels)
        self.bilateral = Lattice(image, None, True, theta_alpha, theta_beta, 1.0, max_channels=n_labels)
        self.spatial = Lattice(None, shape, False, 1.0, 1.0, theta_gamma, max_channels=n_labels)
        if checkpoint not in (None, "8bit"):
            raise ValueError('checkpoint must be None or "8bit"')
        self.checkpoint = checkpoint
        self.bilateral_weight = self._weight(bilateral_weight, "bilateral_weight", image.device)
        self.spatial_weight = self._weight(spatial_weight, "spatial_weight", image.device)
        self.label_bias = None if label_bias is None else self._parameter(label_bias, image.device)
        if label_bias is not None and tuple(label_bias.shape) != (self.n_labels,):
            raise ValueError("label_bias must be [n_labels]")
        # None: Potts model (1 - identity), which the kernel evaluates without the L x L product
        self.compatibility = None if compatibility is None else self._parameter(compatibility, image.device)
        if self.compatibility is not None and tuple(self.compatibility.shape) != (self.n_labels, self.n_labels):
            raise ValueError("compatibility must be [n_labels, n_labels]")

    def _weight(self, w, name, device):
        """A number where nothing can be learned, else a tensor of one value or [n_labels]."""
        if not isinstance(w, torch.Tensor) or (w.numel() == 1 and not w.requires_grad):
            return float(w)
        if tuple(w.shape) not in ((), (1,), (self.n_labels,)):
            raise ValueError("%s must be a number, or a tensor of one value or [n_labels]" % name)
        return self._parameter(w, device)

    @staticmethod
    def _parameter(t, device):
        """What to keep of a tensor: one that is learned as it was given, since a copy would not follow its optimizer; a constant
        as the kernels take it."""
        return t if t.requires_grad else DenseCRF._as_taken(t, device)

    @staticmethod
    def _as_taken(t, device):
        """A kept parameter as the kernels take it: whether or not it is still learned."""
        return t.to(device=device, dtype=torch.float32).contiguous()

    def _by_channel_mix(self):
        """Whether a step has parameters that pl_crf_update_f32 does not take, or has to know their gradients."""
        return isinstance(self.bilateral_weight, torch.Tensor) or isinstance(self.spatial_weight, torch.Tensor) or (
            self.label_bias is not None) or (
            torch.is_grad_enabled() and self.compatibility is not None and self.compatibility.requires_grad)

    def _potts(self, device):
        return 1.0 - torch.eye(self.n_labels, device=device)

    def _mix_weights(self, device):
        """What a step's `channel_mix` multiplies the filtered distributions with, minus weight times compatibility, and its bias."""
        compatibility = self._potts(device) if self.compatibility is None else self._as_taken(self.compatibility, device)
        return tuple(-(self._as_taken(w, device).reshape(-1, 1) if isinstance(w, torch.Tensor) else w) * compatibility
                     for w in (self.bilateral_weight, self.spatial_weight)) + (
                         None if self.label_bias is None else self._as_taken(self.label_bias, device),)

    def step(self, q, unaries):
        """Q after one mean-field update."""
        return self._step(q, unaries, None)

    def _step(self, q, unaries, mix_weights):
        """mix_weights: those of _mix_weights where the caller has them already."""
        grad = torch.is_grad_enabled()
        if self._by_channel_mix():
            self._check_step(q, unaries)
            wb, ws, bias = self._mix_weights(q.device) if mix_weights is None else mix_weights
            if grad and q.requires_grad:
                qb, qs = (_LatticeApplyFunction.apply(lattice, q) for lattice in (self.bilateral, self.spatial))
            else:
                qb, qs = self.bilateral.apply(q), self.spatial.apply(q)
            return channel_mix(qb, wb, bias, unaries, qs, ws, "softmax", -1.0, self.checkpoint)
        if grad and (q.requires_grad or unaries.requires_grad):
            self._check_step(q, unaries)
            return _CrfStepFunction.apply(self, q, unaries)
        return self._constant_step(q, unaries)

    def _check_step(self, q, unaries):
        if q.shape[-1] != self.n_labels or unaries.shape != q.shape:
            raise ValueError("q and unaries must be [B, *S, n_labels]")
        if unaries.dtype != torch.float32 or not unaries.is_cuda:
            raise TypeError("unaries must be a float32 CUDA tensor")

    def _constant_step(self, q, unaries):
        self._check_step(q, unaries)
        unaries = unaries.contiguous()
        if self.compatibility is None:
            out = self._fused_step(q, unaries)
            if out is not None:
                return out
        qb = self.bilateral.apply(q)
        qs = self.spatial.apply(q)
        out = torch.empty_like(qb)
        n_points = out.numel() // self.n_labels
        compatibility = None if self.compatibility is None else self._as_taken(self.compatibility, out.device)
        with torch.cuda.device(out.device):
            capi.check(capi.lib().pl_crf_update_f32(
                out.data_ptr(), unaries.data_ptr(), qb.data_ptr(), qs.data_ptr(),
                0 if compatibility is None else compatibility.data_ptr(), self.bilateral_weight, self.spatial_weight,
                n_points, self.n_labels, _stream_handle(out.device)), "pl_crf_update_f32")
        return out

    def _fused_step(self, q, unaries):
        """The whole step by pl_crf_step_f32, or None where that takes another number of dimensions or labels."""
        a, s = self.bilateral, self.spatial
        call = a.call
        if a.workspace is None or s.workspace is None:
            return None
        _check_tensor(q, "input_image")
        _float32_only(q, "Lattice (build once, apply many times)")
        if tuple(q.shape[:-1]) != (call.batch,) + tuple(call.sdims):
            raise ValueError("input_image does not have the lattice's batch and spatial shape")
        q = q.contiguous()
        out = torch.empty_like(q)
        with _OnDevice(a.device):
            rc = capi.lib().pl_crf_step_f32(
                out.data_ptr(), q.data_ptr(), unaries.data_ptr(), self.bilateral_weight, self.spatial_weight,
                self.n_labels, call.batch, len(call.sdims), call.c_sdims, call.r, a.workspace.data_ptr(),
                a.workspace.numel(), a.max_entries, s.workspace.data_ptr(), s.workspace.numel(), s.max_entries,
                _stream_handle(a.device))
        if rc == capi.PL_UNSUPPORTED_DIMS:
            return None
        capi.check(rc, "pl_crf_step_f32")
        return out

    @staticmethod
    def _start(unaries):
        """softmax(-unaries), zeros where every label is forbidden, in one kernel where pl_crf_start_f32 takes them and torch
        does not follow them: a tracer, a transform or a tensor of another class would not see the kernel, torch's operations
        they do."""
        if type(unaries) not in (torch.Tensor, torch.nn.Parameter) or _watched_by_torch() or not unaries.is_cuda \
                or unaries.dtype != torch.float32 or unaries.dim() < 1 or not 1 <= unaries.shape[-1] <= 128:
            nothing = torch.isposinf(unaries).all(-1, keepdim=True)
            return torch.softmax(-unaries.masked_fill(nothing, 0.0), dim=-1).masked_fill(nothing, 0.0)
        if torch.is_grad_enabled() and unaries.requires_grad:
            return _CrfStartFunction.apply(unaries)
        return _start_kernel(unaries)

    def infer(self, unaries, iterations=5):
        """Q after `iterations` mean-field updates, starting from softmax(-unaries)."""
        q = self._start(unaries)
        mix_weights = self._mix_weights(unaries.device) if self._by_channel_mix() else None   # once, not in every step
        for _ in range(int(iterations)):
            q = self._step(q, unaries, mix_weights)
        return q


def _main():
    """python -m permutohedral_lattice_b200.crf [--batch B] [--size S] [--labels L] [--iterations K] [--train] [--checkpoint 8bit]
    Times mean-field iterations on the synthetic dense-CRF workload (seeded; no dataset belongs to this path); with --train
    an inference of K iterations and its gradients (unaries, kernel weights, compatibility, label bias)."""
    import argparse

    from . import workloads
    ap = argparse.ArgumentParser()
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--size", type=int, default=512)
    ap.add_argument("--labels", type=int, default=21)
    ap.add_argument("--iterations", type=int, default=10)
    ap.add_argument("--train", action="store_true")
    ap.add_argument("--checkpoint", choices=["8bit"])
    args = ap.parse_args()
    w = workloads.config2(batch=args.batch, size=args.size, channels=args.labels)
    image = torch.from_numpy(w.reference).cuda()
    q0 = torch.from_numpy(w.input).cuda()
    unaries = -torch.log(q0 + 1e-6)
    if args.train:
        return _time_training(args, w, image, unaries)
    crf = DenseCRF(image, args.labels, w.theta_alpha, w.theta_beta, 3.0)
    q = q0
    for _ in range(3):
        q = crf.step(q, unaries)
    torch.cuda.synchronize()
    t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    t0.record()
    for _ in range(args.iterations):
        q = crf.step(q, unaries)
    t1.record()
    torch.cuda.synchronize()
    ms = t0.elapsed_time(t1) / args.iterations
    print("%d x %dx%d, %d labels: %.3f ms per mean-field iteration (two lattice applications + fused update), "
          "%.1f Mpixels/s" % (args.batch, args.size, args.size, args.labels, ms,
                             args.batch * args.size * args.size / ms / 1e3))


def _time_training(args, w, image, unaries):
    labels = args.labels
    params = [torch.ones(labels, device="cuda", requires_grad=True) for _ in range(2)] + [
        (1.0 - torch.eye(labels, device="cuda")).requires_grad_(True), torch.zeros(labels, device="cuda", requires_grad=True)]
    crf = DenseCRF(image, labels, w.theta_alpha, w.theta_beta, 3.0, *params, checkpoint=args.checkpoint)
    unaries.requires_grad_(True)
    grad = torch.randn_like(unaries)

    def pass_():
        return torch.autograd.grad(crf.infer(unaries, args.iterations), [unaries] + params, grad)

    pass_()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    t0.record()
    for _ in range(3):
        pass_()
    t1.record()
    torch.cuda.synchronize()
    ms = t0.elapsed_time(t1) / 3
    print("%d x %dx%d, %d labels, %d iterations%s: %.3f ms an inference with its gradients, %.1f Mpixels/s an iteration, "
          "%.2f GB beside inputs and lattices" % (
              args.batch, args.size, args.size, labels, args.iterations, ", 8 bits" if args.checkpoint else "", ms,
              args.batch * args.size * args.size * args.iterations / ms / 1e3,
              (torch.cuda.max_memory_allocated() - before) / 1e9))


if __name__ == "__main__":
    _main()
