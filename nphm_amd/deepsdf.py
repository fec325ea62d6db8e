"""Host-side mirror of the reference's global DeepSDF and forward-deformation network
(src/NPHM/models/deepSDF.py): same class names, constructor signatures, attributes, ``forward``
contracts and ``state_dict`` layout (``lin{i}.{weight,bias}``, ``compressor.0.*``,
``defDeepSDF.lin{i}.*``).

Execution tiers (same policy as the identity field, ensembled_deepsdf.py):

* **HIP** (``libnphm_amd.so``, gfx950): whenever no autograd graph is needed, the tensors live on a
  ROCm device, the architecture is covered (``nphm_mlp_supported``: the NPM net and the NPHM
  deformation backbone are) and the conditioning is constant along the point axis.  One fused
  kernel runs the whole skip-MLP; if the library is missing this tier raises.
* **composite**: ``DeepSDF.evaluate`` — a differentiable PyTorch formulation in which the latent
  columns of the first layer and of the skip layer are applied once per latent row.  Used when
  gradients are required, for per-point conditioning (training-mode noise, 'interpolate') and for
  other architectures.  Never chosen silently on a CPU tensor: that needs ``backend = "composite"``.
"""
from __future__ import annotations

import math
from contextlib import contextmanager
from typing import Optional

import os

import numpy as np
import torch
import torch.nn as nn

from . import _lib
from .train_ops import grad_norm, linear_act
from .ensembled_deepsdf import sample_point_feature  # noqa: F401  (re-exported like the reference)

_SQRT2 = float(np.sqrt(2))


class _MlpCondFn(torch.autograd.Function):
    """out = mlp(xyz; cond_rows) with the fused forward kernel and a hand-written first-order backward with respect
    to the CONDITIONING rows (mlp_bwd_kernel.hip): what the fitting loop differentiates through the deformation
    field (fitting.py:99-106; the query points are detached roots, the decoder is frozen).  The forward leaves
    sigma' of every hidden layer in a scratch buffer; the backward kernel returns the bias gradients of lin0 and of
    the skip layer, which the two latent blocks of those layers map onto the conditioning vector."""

    @staticmethod
    def forward(ctx, module, xyz, cond_rows, add_input, with_jacobian=False, with_inverse=False, implicit_root=False):
        """-> [R,n,out] or, ``with_jacobian``, (value [R,n,out], [R,n,3,out] = d/dx | d/dy | d/dz as forward_hip_jvp; only
        the value is differentiable) - and, ``with_inverse``, the inverse [R,n,3,3] of the Jacobian of the first three
        outputs (rows = outputs, columns = x, y, z) from the same launch.
        ``implicit_root`` (with ``add_input``, jacobian and inverse; out_dim 3): ``xyz`` are roots of x + F(x; cond) = obs and
        the FIRST output is  x_c = xyz - J^-1 (F - F.detach())  (fitting.py:99-106): the roots themselves, whose gradient
        reaches the conditioning through -J^-T - applied by the backward kernel while it loads the gradient"""
        lib = _lib.load()
        R, n, _ = xyz.shape
        dev = xyz.device
        packed, state = module.prepare_latent(cond_rows.detach())
        xyz_c = xyz.detach().contiguous().float()
        saved = torch.empty(lib.nphm_mlp_saved_bytes(*module._arch(), R, n), dtype=torch.uint8, device=dev)
        stream = torch.cuda.current_stream(dev).cuda_stream
        code = module._fit_code(packed, state, xyz_c)
        jinv = None
        if with_jacobian:
            out = torch.empty(R, n, 4, module.n_out, dtype=torch.float32, device=dev)
            if with_inverse:
                jinv = torch.empty(R, n, 3, 3, dtype=torch.float32, device=dev)
            for p0, cnt, cols in module._jvp_split(R, n, dev, 64):
                _lib.check(lib.nphm_mlp_eval_points_jvp_saving(*module._arch(), packed.data_ptr(), state.data_ptr(),
                                                               xyz_c.data_ptr(), R, n, int(bool(add_input)), out.data_ptr(),
                                                               saved.data_ptr(), code, p0, cnt, cols,
                                                               None if jinv is None else jinv.data_ptr(), stream),
                           "nphm_mlp_eval_points_jvp_saving")
        else:
            out = torch.empty(R, n, module.n_out, dtype=torch.float32, device=dev)
            _lib.check(lib.nphm_mlp_eval_points_saving(*module._arch(), packed.data_ptr(), state.data_ptr(), xyz_c.data_ptr(),
                                                       R, n, int(bool(add_input)), out.data_ptr(), saved.data_ptr(), code, stream),
                       "nphm_mlp_eval_points_saving")
        ctx.module, ctx.shape, ctx.with_jacobian = module, (R, n), bool(with_jacobian)
        ctx.root = bool(implicit_root)
        if ctx.root:
            assert jinv is not None and add_input and module.n_out == 3, "implicit root: value + Jacobian + inverse of a 3-vector field"
            ctx.save_for_backward(saved, jinv)
            ctx.set_materialize_grads(False)
            jac = out[:, :, 1:]
            root = xyz_c.view(R, n, 3).detach()
            ctx.mark_non_differentiable(jac, jinv)
            return root, jac, jinv
        ctx.save_for_backward(saved)
        if not with_jacobian:
            return out
        # value and Jacobian as TWO outputs (views of the kernel's interleaved buffer): the value's gradient then arrives
        # as its own tensor - a single output would receive zeros [R,n,4,out] + a slice copy from autograd, and the
        # backward below would copy the slice out again
        jac = out[:, :, 1:]
        ctx.set_materialize_grads(False)       # (no zeros [R,n,3,out] + fill launch for the Jacobian's absent gradient)
        if jinv is not None:
            ctx.mark_non_differentiable(jac, jinv)
            return out[:, :, 0], jac, jinv
        ctx.mark_non_differentiable(jac)
        return out[:, :, 0], jac

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out, _grad_jac=None, _grad_jinv=None):
        if grad_out is None:
            return None, None, None, None, None, None, None
        lib = _lib.load()
        module = ctx.module
        saved, *rest = ctx.saved_tensors
        root_jinv = rest[0] if ctx.root else None
        R, n = ctx.shape
        dev = grad_out.device
        H = module.hidden_dim
        # per 32-point slot of every row the bias gradients of lin0 | the skip layer (every slot written: no zero fill)
        parts = torch.empty(lib.nphm_mlp_bwd_partial_bytes(H, R, n) // 4, dtype=torch.float32, device=dev)
        g = grad_out.detach().contiguous().float()
        stream = torch.cuda.current_stream(dev).cuda_stream
        _lib.check(lib.nphm_mlp_backward_cond(*module._arch(), module._packed_bwd(dev).data_ptr(), saved.data_ptr(),
                                              g.data_ptr(), None if root_jinv is None else root_jinv.data_ptr(), R, n, parts.data_ptr(), stream),
                   "nphm_mlp_backward_cond")
        d = module.input_dim
        skip = module.skip_in[0]
        W0 = module.lin0.weight                                   # [H, d + lat]
        Ws = getattr(module, f"lin{skip}").weight                 # [H, k_act + d + lat]
        k_act = Ws.shape[1] - W0.shape[1]
        lat = W0.shape[1] - d
        if W0.dtype == torch.float32 and W0.is_contiguous() and Ws.is_contiguous():
            # gb0 W0[:, d:] + gbs Ws[:, k_act + d:] / sqrt2 in one launch (two library GEMMs on 5 rows, a divide, an add)
            grad_cond = torch.empty(R, lat, dtype=torch.float32, device=dev)
            _lib.check(lib.nphm_mlp_cond_grad(parts.data_ptr(), n, R, H, W0.detach().data_ptr(), W0.shape[1], d,
                                              Ws.detach().data_ptr(), Ws.shape[1], k_act + d, lat, grad_cond.data_ptr(), stream),
                       "nphm_mlp_cond_grad")
        else:
            gb0, gbs = parts.view(R, -1, 2, H).sum(dim=1).unbind(1)
            grad_cond = gb0 @ W0[:, d:] + (gbs @ Ws[:, k_act + d:]) / _SQRT2
        return None, None, grad_cond, None, None, None, None


class _DenseLayerFn(torch.autograd.Function):
    """y = act(alpha x W^T + b) of one nn.Linear (+ Softplus) of the backbone with TRAINABLE parameters, on the kernels of
    csrc/dense_train_kernels.hip: one launch forward; backward: act' from y and the transposes (one launch + two small ones),
    dx = alpha gp W (one launch), dW = alpha gp^T x with the point axis as K in splits added in order (two launches), db = column
    sums of gp (per 32-row tile in the first launch, one more over the tiles).  First order only.  x [M,K], W [N,K], b [N]; beta None: no activation."""

    @staticmethod
    def forward(ctx, x, weight, bias, alpha, beta):
        lib = _lib.load()
        x = x.contiguous()
        W = weight.detach().contiguous()
        M, K = x.shape
        N = W.shape[0]
        y = torch.empty(M, N, dtype=torch.float32, device=x.device)
        stream = torch.cuda.current_stream(x.device).cuda_stream
        b = bias.detach().contiguous()
        _lib.check(lib.nphm_dense_gemm_nt(x.data_ptr(), K, W.data_ptr(), K, y.data_ptr(), N, M, N, K, b.data_ptr(), M,
                                          float(alpha), 0.0 if beta is None else float(beta), 2 if beta is None else 1, 1, stream),
                   "nphm_dense_gemm_nt")
        ctx.save_for_backward(x, W, y)
        ctx.alpha, ctx.beta = float(alpha), beta
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        lib = _lib.load()
        x, W, y = ctx.saved_tensors
        M, K = x.shape
        N = W.shape[0]
        dev = x.device
        stream = torch.cuda.current_stream(dev).cuda_stream
        pad4 = lambda v: (v + 3) // 4 * 4
        g = g.contiguous()
        ldm = pad4(M)
        gp = torch.empty(M, N, dtype=torch.float32, device=dev)
        gp_t = torch.empty(N, ldm, dtype=torch.float32, device=dev)
        tiles = torch.empty((M + 31) // 32, N, dtype=torch.float32, device=dev) if ctx.needs_input_grad[2] else None
        _lib.check(lib.nphm_dense_gpre(g.data_ptr(), None if ctx.beta is None else y.data_ptr(), M, N,
                                       0.0 if ctx.beta is None else float(ctx.beta), gp.data_ptr(), gp_t.data_ptr(), ldm,
                                       None if tiles is None else tiles.data_ptr(), stream), "nphm_dense_gpre")
        dx = dW = db = None
        if ctx.needs_input_grad[0]:
            ldn = pad4(N)
            w_t = torch.empty(K, ldn, dtype=torch.float32, device=dev)
            _lib.check(lib.nphm_dense_gpre(W.data_ptr(), None, N, K, 0.0, None, w_t.data_ptr(), ldn, None, stream), "nphm_dense_gpre")
            dx = torch.empty(M, K, dtype=torch.float32, device=dev)
            _lib.check(lib.nphm_dense_gemm_nt(gp.data_ptr(), N, w_t.data_ptr(), ldn, dx.data_ptr(), K, M, K, N, None, 1,
                                              ctx.alpha, 0.0, 0, 1, stream), "nphm_dense_gemm_nt")
        if ctx.needs_input_grad[1]:
            x_t = torch.empty(K, ldm, dtype=torch.float32, device=dev)
            _lib.check(lib.nphm_dense_gpre(x.data_ptr(), None, M, K, 0.0, None, x_t.data_ptr(), ldm, None, stream), "nphm_dense_gpre")
            splits = int(min(64, max(1, M // 512)))
            parts = torch.empty(splits, N, K, dtype=torch.float32, device=dev)
            _lib.check(lib.nphm_dense_gemm_nt(gp_t.data_ptr(), ldm, x_t.data_ptr(), ldm, parts.data_ptr(), K, N, K, M, None, 1,
                                              1.0, 0.0, 0, splits, stream), "nphm_dense_gemm_nt")
            dW = torch.empty(N, K, dtype=torch.float32, device=dev)
            _lib.check(lib.nphm_dense_reduce_splits(parts.data_ptr(), splits, N * K, ctx.alpha, dW.data_ptr(), stream),
                       "nphm_dense_reduce_splits")
        if ctx.needs_input_grad[2]:
            db = torch.empty(N, dtype=torch.float32, device=dev)
            _lib.check(lib.nphm_dense_column_sums(tiles.data_ptr(), tiles.shape[0], N, db.data_ptr(), stream), "nphm_dense_column_sums")
        return dx, dW, db, None, None


class _GemmNTFn(torch.autograd.Function):
    """C = alpha A B^T on nphm_dense_gemm_nt (split-bf16 x3 MFMA, fp32 accumulate), differentiable to ANY order: its backward
    is made of the same product (dA = alpha G B = gemm(G, B^T), dB = alpha G^T A = gemm(G^T, A^T); the transposes are torch
    copies) - what the second-order passes of loss_joint / the NPM trainer (``gradient(sdf, x, create_graph=True)``, then
    ``backward()``) need, which the fused first-order ``_DenseLayerFn`` cannot serve.  A [M,K], B [N,K] fp32 on a ROCm device."""

    @staticmethod
    def forward(ctx, A, B, alpha):
        lib = _lib.load()
        if not (A.is_contiguous() and B.is_contiguous()):
            raise ValueError("_GemmNTFn: contiguous operands (copy OUTSIDE the function: a saved copy made here is detached)")
        M, K = A.shape
        N = B.shape[0]
        dev = A.device
        stream = torch.cuda.current_stream(dev).cuda_stream
        C = torch.empty(M, N, dtype=torch.float32, device=dev)
        splits = int(min(64, K // 1024)) if (K >= 4096 and (M + 127) // 128 * ((N + 255) // 256) < 128) else 1
        if splits > 1:       # a long K over a small result (a weight gradient): ordered splits fill the chip
            parts = torch.empty(splits, M, N, dtype=torch.float32, device=dev)
            _lib.check(lib.nphm_dense_gemm_nt(A.data_ptr(), K, B.data_ptr(), K, parts.data_ptr(), N, M, N, K, None, 1, 1.0, 0.0, 0, splits,
                                              stream), "nphm_dense_gemm_nt")
            _lib.check(lib.nphm_dense_reduce_splits(parts.data_ptr(), splits, M * N, float(alpha), C.data_ptr(), stream),
                       "nphm_dense_reduce_splits")
        else:
            _lib.check(lib.nphm_dense_gemm_nt(A.data_ptr(), K, B.data_ptr(), K, C.data_ptr(), N, M, N, K, None, 1, float(alpha), 0.0, 0, 1,
                                              stream), "nphm_dense_gemm_nt")
        ctx.save_for_backward(A, B)
        ctx.alpha = float(alpha)
        return C

    @staticmethod
    def backward(ctx, G):
        A, B = ctx.saved_tensors
        dA = dB = None
        G = G.contiguous()
        if ctx.needs_input_grad[0]:
            dA = _GemmNTFn.apply(G, B.t().contiguous(), ctx.alpha)
        if ctx.needs_input_grad[1]:
            dB = _GemmNTFn.apply(G.t().contiguous(), A.t().contiguous(), ctx.alpha)
        return dA, dB, None


# Gradients between layers in fp16.  A mean over thousands of points leaves entries of 1e-7 and less, most of which fp16 holds as zero or with a few
# bits.  The gradient that enters a run of 16-bit layers is therefore raised by a power of two where its largest entry is below 2^-8, and
# what leaves the run (towards the layer in front, the weights and the biases) is lowered by the same one.  The largest entry goes to 2^9 .. 2^10
# over the number of rows: a weight's gradient adds that many products, and 2^6 are left to fp16's end for what the layers
# multiply it by.  Larger gradients pass as they are.  Nothing waits for the device.
_FP16_SMALL, _FP16_ROOM = 2.0 ** -8, 10


class _LeaveHalf(torch.autograd.Function):
    """x in fp32; its gradient, raised, in x's type.  run: a list that takes the power of two"""

    @staticmethod
    def forward(ctx, x, run):
        ctx.run, ctx.dtype = run, x.dtype
        return x.float()

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        top = grad_norm([g], float("inf"))
        up = _FP16_ROOM - max(g.shape[0] - 1, 0).bit_length() - torch.frexp(top).exponent
        up = torch.where((top > 0) & (top < _FP16_SMALL), up.clamp(0, 126), torch.zeros_like(up))        # (no number: left alone)
        ctx.run[:] = [(up + 127 << 23).to(torch.int32).view(torch.float32).view(1)]
        return (g * ctx.run[0]).to(ctx.dtype), None


class _EnterHalf(torch.autograd.Function):
    """The tensors of a run (its first input, the weights and biases) in fp16; their gradients in fp32, lowered by what ``_LeaveHalf`` at the
    other end has raised them by.  One node for all of them (with one each a step of 5000 points through six layers of 512 took 1.39 ms, 1.27 so).
    What asks for no gradient is passed on without."""

    @staticmethod
    def forward(ctx, run, *tensors):
        ctx.run = run
        ctx.set_materialize_grads(False)
        out = tuple(t.half() for t in tensors)
        ctx.mark_non_differentiable(*[h for h, asks in zip(out, ctx.needs_input_grad[1:]) if not asks])
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        return (None, *[None if g is None else g / ctx.run[0] for g in grads])         # (a [1] of fp32: the quotient is fp32)


class DeepSDF(nn.Module):
    """Skip-MLP SDF / vector field (deepSDF.py:6-89).  dims = [d_in] + [hidden]*nlayers + [out];
    the input is re-injected (concatenated, divided by sqrt 2) before layer ``nlayers//2``;
    Softplus(beta) activations (ReLU if beta <= 0); optional geometric init of the last layer."""

    # storage of the dense training tier's hidden layers: "fp32", or "bf16" | "fp16" (train_ops.linear_act) for the layers that
    # read hidden values alone; the layers that read coordinates (the first, the skip layer) and the last stay in fp32 -
    # a coordinate of 0.5 would move by up to 1e-3 in bf16.  Gradients between fp16 layers are scaled where fp16 would lose them.
    # (On the class: modules pickled whole without it still train.)
    train_precision = "fp32"

    def __init__(self, lat_dim, hidden_dim, nlayers=8, geometric_init=True, radius_init=1, beta=100,
                 out_dim=1, num_freq_bands=None, input_dim=3):
        super().__init__()
        d_spatial = input_dim if num_freq_bands is None else input_dim * (2 * num_freq_bands + 1)
        d_in = lat_dim + d_spatial
        self.lat_dim = lat_dim
        self.input_dim = input_dim
        self.d_spatial = d_spatial
        self.hidden_dim = hidden_dim
        self.nlayers = nlayers
        self.n_out = out_dim
        self.beta = beta
        self.backend = "hip"            # "hip" | "composite"
        self.train_backend = "hip"      # with trainable parameters: "hip" = the dense training tier (evaluate_train_hip) | "composite"
        self._pack_cache = None         # (key, packed tensor)
        self._pack_bwd_cache = None     # (key, transposed pack of the backward kernel)
        # Numerics of the plain HIP evaluation (forward_hip / lattice launches; include/nphm_amd.h NPHM_MLP_*):
        #   precision "f16x3" (default) | "bf16x3": operand format of the split products;
        #   numerics "auto": on evaluations of >= two_pass_min_points points the cheapest tier whose output stays within
        #   `numerics_target` of the three-term product on a sample (calibrate_numerics / _numerics_code below; verified on a
        #   sample of every such call): per hidden layer the single-term product rn(x) wh (split-f16 only; in EVERY layer:
        #   twice the points per weight pass), the two-term product xh wh + xl wh, or all three terms;
        #   "fixed": exactly `single_mask` / `two_pass_mask` (0 / 0 = the three-term product everywhere).
        self.precision = os.environ.get("NPHM_AMD_MLP_PRECISION", "f16x3")
        self.numerics = os.environ.get("NPHM_AMD_MLP_NUMERICS", "auto")
        self.two_pass_mask = 0
        self.single_mask = 0            # ("fixed") hidden layers on the single-term product; all of them: 128 points per workgroup
        # max |tier - three-term| allowed on the calibration / verification sample (output units).  5e-6 = the bar of the
        # identity field's calibrated tiers (numerics.py); rounds 3-4 used 2e-6 here, which the two-term tier meets
        # (0.7 - 1.3e-6 on the seeded and trained-like nets) and the single-term tier misses by a hair (2.1e-6)
        self.numerics_target = float(os.environ.get("NPHM_AMD_MLP_TARGET", "5e-6"))
        self.allow_single_term = os.environ.get("NPHM_AMD_MLP_SINGLE", "1") not in ("0", "")
        # the tier set "single-term everywhere, last hidden layer two-term" with a workspace (eval_workspace): that layer's
        # weights streamed once (two K halves) instead of twice (two point halves); same bits either way.  Opt-in: measured
        # 11.6 % fewer L2 requests, the same time (4.187 / 4.195 ms) and 1.1 GB more HBM-side traffic per launch for the
        # parked halves - the workspace-free form stays the default
        self.tail_k_split = os.environ.get("NPHM_AMD_MLP_TAIL_KSPLIT", "0") not in ("0", "")
        self.two_pass_min_points = 1 << 18
        self._two_pass_cache = None     # (weight key, calibrated mask, report)
        # The value+Jacobian / Broyden / gradient-saving launches (the correspondence search and the implicit differentiation
        # of a fitting step: 5 000 points, weights frozen, conditioning moving with the codes): "auto" = split-f16 operands
        # with the two-term layers of a mask calibrated ONCE per weight version (first such call outside a stream capture, on
        # a sample of its points and its first conditioning row; nothing can be re-measured inside the replayed graph) |
        # "f16x3" | "bf16x3" (rounds 1-3): three terms everywhere
        self.fit_numerics = os.environ.get("NPHM_AMD_FIT_NUMERICS", "auto")
        self.fit_target = 2e-6          # bound on the value of those launches (two-term against three-term), output units
        self.fit_jacobian_target = 2e-5  # ... and on their Jacobian entries
        self.fit_verify_every = 100     # fitting steps between two re-measurements on the current codes (reverify_fit)
        self._fit_cache = None          # (weight key, mask, report)
        self._fit_last = None
        self.last_numerics = None       # what the most recent large evaluation ran (for bench.py / diagnostics)
        self._state_scope = None        # inside DeformationNetwork.condition_scope(): {cond tensor key: (tensor, state)}
        print(d_in)
        print(hidden_dim)
        dims = [d_in] + [hidden_dim] * nlayers + [out_dim]
        self.num_layers = len(dims)
        self.skip_in = [nlayers // 2]
        self.num_freq_bands = num_freq_bands
        if num_freq_bands is not None:
            self.freq_bands = 2 ** torch.arange(num_freq_bands)
        for layer in range(self.num_layers - 1):
            fan_out = dims[layer + 1] - d_in if (layer + 1) in self.skip_in else dims[layer + 1]
            lin = nn.Linear(dims[layer], fan_out)
            if geometric_init and layer == self.num_layers - 2:
                nn.init.normal_(lin.weight, mean=np.sqrt(np.pi) / np.sqrt(dims[layer]), std=0.00001)
                nn.init.constant_(lin.bias, -radius_init)
            setattr(self, f"lin{layer}", lin)
        self.activation = nn.Softplus(beta=beta) if beta > 0 else nn.ReLU()

    def _embed(self, xyz):
        if self.num_freq_bands is None:
            return xyz
        parts = [xyz]
        for freq in self.freq_bands:
            parts.append(torch.sin(xyz * freq))
            parts.append(torch.cos(xyz * freq))
        return torch.cat(parts, dim=-1)

    @property
    def two_pass_target(self):
        """(rounds 3-4 name of ``numerics_target``)"""
        return self.numerics_target

    @two_pass_target.setter
    def two_pass_target(self, v):
        self.numerics_target = float(v)

    def evaluate(self, pos, lat, gemm_hip=False):
        """pos [B,N,d_spatial]; lat [B,Lr,lat_dim], Lr in {1,N}.  ``gemm_hip``: the hidden x W^T products (M = B N rows) on
        ``_GemmNTFn`` instead of a library GEMM - same op sequence, differentiable to any order."""
        D = pos.shape[-1]
        last = self.num_layers - 2
        x = None
        # (operands made contiguous OUT HERE, by differentiable copies: a copy made inside the Function would be saved detached,
        # and the second-order term that reaches a weight through d/dx = G W would be lost - the skip layer's column slice)
        mm = (lambda a, w: _GemmNTFn.apply(a.reshape(-1, a.shape[-1]).contiguous(), w.contiguous(), 1.0).reshape(*a.shape[:-1], w.shape[0])) \
            if gemm_hip else (lambda a, w: a @ w.t())
        for layer in range(self.num_layers - 1):
            lin = getattr(self, f"lin{layer}")
            W, b = lin.weight, lin.bias
            if layer == 0 or layer in self.skip_in:
                n_prev = 0 if layer == 0 else x.shape[-1]
                scale = 1.0 if layer == 0 else 1.0 / _SQRT2
                lat_term = (lat @ W[:, n_prev + D:].t()) * scale + b          # [B,Lr,out]
                y = (pos @ W[:, n_prev:n_prev + D].t()) * scale
                if layer != 0:
                    y = y + mm(x, W[:, :n_prev]) * scale
                x = y + lat_term
            elif layer < last:
                x = mm(x, W) + b
            else:
                x = x @ W.t() + b
            if layer < last:
                x = self.activation(x)
        return x

    def train_tier_serves(self, xyz, lat):
        """The dense training tier's conditions: trainable parameters, a recorded graph, ROCm fp32 tensors, and no gradient
        asked w.r.t. the query points (its backward is first order: loss_joint's d sdf / d posed points through the offsets
        needs the composite tier's double backward)."""
        return (self.backend != "composite" and self.train_backend == "hip" and xyz.is_cuda and xyz.dtype == torch.float32
                and lat.dtype == torch.float32 and torch.is_grad_enabled() and not xyz.requires_grad
                and any(p.requires_grad for p in self.parameters())
                and all(p.dtype == torch.float32 for p in self.parameters()))

    def gemm_tier_serves(self, xyz, lat):
        """The any-order tier: a recorded graph on ROCm fp32 tensors with enough rows to fill the chip (``evaluate`` with its
        hidden products on ``_GemmNTFn``) - what serves a call the first-order training tier cannot (a gradient w.r.t. the
        query points that is differentiated again)."""
        return (self.backend != "composite" and self.train_backend == "hip" and xyz.is_cuda and xyz.dtype == torch.float32
                and lat.dtype == torch.float32 and torch.is_grad_enabled() and xyz.shape[0] * xyz.shape[1] >= 2048
                and (xyz.requires_grad or lat.requires_grad or any(p.requires_grad for p in self.parameters()))
                and all(p.dtype == torch.float32 for p in self.parameters()))

    def evaluate_train_hip(self, pos, lat):
        """``evaluate`` with every hidden nn.Linear + activation as ONE launch of csrc/dense_train_kernels.hip and its
        backward - data, weight and bias gradients - on the same kernels (``_DenseLayerFn``): the op sequence of the reference's
        forward (deepSDF.py:64-89: cat, skip cat / sqrt 2, Linear, Softplus), the concatenations left to torch.  With ``train_precision``
        "bf16" or "fp16" the layers between run in 16-bit storage (``linear_act``).  The last
        linear layer (out_dim <= 4 rows) stays an nn.Linear call.  pos [B,N,d_spatial]; lat [B,Lr,lat_dim], Lr in {1,N}."""
        B, N, _ = pos.shape
        lat_full = lat if lat.shape[1] == N else lat.expand(B, N, lat.shape[-1])
        inp = torch.cat([pos, lat_full], dim=-1).reshape(B * N, -1)
        x = inp
        last = self.num_layers - 2
        beta = float(self.beta)
        try:
            half = {"fp32": None, "bf16": torch.bfloat16, "fp16": torch.float16}[self.train_precision]
        except KeyError:
            raise ValueError(f"train_precision is 'fp32', 'bf16' or 'fp16', not {self.train_precision!r}") from None
        within = [half is not None and 0 < k < last and k not in self.skip_in for k in range(last + 1)]
        run, params = [], {}                        # fp16: the scale of the gradients in a run of 16-bit layers, its parameters in fp16
        for layer in range(self.num_layers - 1):
            lin = getattr(self, f"lin{layer}")
            alpha = 1.0
            if within[layer]:
                if half == torch.float16 and not within[layer - 1]:
                    mine = [getattr(self, f"lin{k}") for k in range(layer, within.index(False, layer))]
                    x, *flat = _EnterHalf.apply(run, x, *[t for m in mine for t in (m.weight, m.bias)])
                    params.update(zip(mine, zip(flat[::2], flat[1::2])))
                w, b = params[lin] if lin in params else (lin.weight.to(half), lin.bias.to(half))
                x = linear_act(x.to(half), w, b, "softplus" if beta > 0 else "relu", max(beta, 1e-6))
                continue
            if x.dtype == torch.float16:
                x, run = _LeaveHalf.apply(x, run), []
            elif half is not None:
                x = x.float()
            if layer in self.skip_in:
                x = torch.cat([x, inp], dim=-1)
                alpha = 1.0 / _SQRT2
            if layer < last:
                x = _DenseLayerFn.apply(x, lin.weight, lin.bias, alpha, beta)
            else:
                x = torch.nn.functional.linear(x * alpha if alpha != 1.0 else x, lin.weight, lin.bias)
        return x.reshape(B, N, -1)

    # ---- HIP tier ----------------------------------------------------------------------------
    def invalidate_pack(self):
        """Drop the cached split-bf16 copy of the weights (see FastEnsembleDeepSDFMirrored.invalidate_pack:
        needed after writes that bypass the parameters' version counters)."""
        self._pack_cache = None
        self._pack_bwd_cache = None
        self._two_pass_cache = None
        self._fit_cache = None

    def load_state_dict(self, *args, **kwargs):
        out = super().load_state_dict(*args, **kwargs)
        self.invalidate_pack()
        return out

    def _apply(self, fn, *args, **kwargs):
        out = super()._apply(fn, *args, **kwargs)
        self.invalidate_pack()
        return out

    def _arch(self):
        return (self.lat_dim, self.hidden_dim, self.nlayers, self.n_out)

    def hip_supported(self) -> bool:
        lib = _lib.load()
        return bool(lib.nphm_mlp_supported(*self._arch(), self.input_dim, float(self.beta),
                                           0 if self.num_freq_bands is None else int(self.num_freq_bands)))

    def _lin_params(self):
        lins = [getattr(self, f"lin{i}") for i in range(self.num_layers - 1)]
        return [m.weight for m in lins], [m.bias for m in lins]

    def _packed(self, device):
        """Split-bf16 MFMA-fragment copy of the weights on ``device``; rebuilt when a parameter
        changed (optimizer step, load_state_dict, .to())."""
        ws, bs = self._lin_params()
        key = tuple((t.data_ptr(), t._version, str(t.device)) for t in ws + bs) + (str(device),)
        if self._pack_cache is not None and self._pack_cache[0] == key:
            return self._pack_cache[1]
        lib = _lib.load()
        for t in ws + bs:
            if t.device != device or t.dtype != torch.float32 or not t.is_contiguous():
                raise _lib.NphmAmdError("DeepSDF parameters must be contiguous fp32 on the query device")
        packed = torch.empty(lib.nphm_mlp_packed_bytes(*self._arch()), dtype=torch.uint8, device=device)
        stream = torch.cuda.current_stream(device).cuda_stream
        _lib.check(lib.nphm_mlp_pack(*self._arch(), _lib.ptr_array(ws), _lib.ptr_array(bs), packed.data_ptr(),
                                     stream), "nphm_mlp_pack")
        self._pack_cache = (key, packed)
        return packed

    def _packed_bwd(self, device):
        """Transposed split-bf16 pack for nphm_mlp_backward_cond (cached like _packed)."""
        ws, _ = self._lin_params()
        key = tuple((t.data_ptr(), t._version, str(t.device)) for t in ws) + (str(device),)
        if self._pack_bwd_cache is not None and self._pack_bwd_cache[0] == key:
            return self._pack_bwd_cache[1]
        lib = _lib.load()
        packed = torch.empty(lib.nphm_mlp_bwd_packed_bytes(*self._arch()), dtype=torch.uint8, device=device)
        stream = torch.cuda.current_stream(device).cuda_stream
        _lib.check(lib.nphm_mlp_pack_bwd(*self._arch(), _lib.ptr_array(ws), packed.data_ptr(), stream), "nphm_mlp_pack_bwd")
        self._pack_bwd_cache = (key, packed)
        return packed

    def hip_backward_supported(self) -> bool:
        return bool(_lib.load().nphm_mlp_bwd_packed_bytes(*self._arch())) and self.hip_supported()

    def forward_hip_cond_grad(self, xyz, cond_rows, add_input=False):
        """``forward_hip`` that is differentiable (first order) with respect to ``cond_rows``."""
        return _MlpCondFn.apply(self, xyz, cond_rows, add_input)

    def prepare_latent(self, cond_rows: torch.Tensor):
        """cond_rows [B, lat_dim] -> (packed weights, per-row state) via the HIP prologue kernel."""
        lib = _lib.load()
        device = cond_rows.device
        packed = self._packed(device)
        key = None
        if self._state_scope is not None:
            # same conditioning tensor again inside one condition_scope (the scope keeps it alive: no address reuse)
            key = (cond_rows.data_ptr(), cond_rows._version, tuple(cond_rows.shape), tuple(cond_rows.stride()))
            hit = self._state_scope.get(key)
            if hit is not None:
                return packed, hit[1]
        cond_in = cond_rows
        cond_rows = cond_rows.contiguous().float()
        B = cond_rows.shape[0]
        state = torch.empty(lib.nphm_mlp_latent_state_bytes(*self._arch(), B), dtype=torch.uint8, device=device)
        ws, bs = self._lin_params()
        stream = torch.cuda.current_stream(device).cuda_stream
        _lib.check(lib.nphm_mlp_prepare_latent(*self._arch(), _lib.ptr_array(ws), _lib.ptr_array(bs),
                                               cond_rows.data_ptr(), B, state.data_ptr(), stream),
                   "nphm_mlp_prepare_latent")
        if key is not None:
            self._state_scope[key] = (cond_in, state)
        return packed, state

    # ---- numerics of the plain evaluation --------------------------------------------------------------------------
    def _format_code(self) -> int:
        if self.precision not in ("f16x3", "bf16x3"):
            raise ValueError(f"DeepSDF.precision must be 'f16x3' or 'bf16x3', got {self.precision!r}")
        return 1 if self.precision == "f16x3" else 0

    def _hidden_mask(self) -> int:
        """Bits of the linear layers that are hidden GEMM layers (1 .. nlayers - 1): the ones a two-term product may serve."""
        return ((1 << self.nlayers) - 1) & ~1

    def eval_workspace(self, code: int, device) -> Optional[torch.Tensor]:
        """Scratch of a plain evaluation launch with the tiers ``code`` (``nphm_mlp_eval_*_ws``), or None where the kernel has
        no use for one.  It serves one tier set: every hidden layer single-term but the last, that one two-term (NPM's) -
        the last hidden layer then streams its weights once, the second K half of its operands waiting in the workspace.
        From torch's caching allocator, per call: stream-ordered like every other temporary, nothing kept alive here."""
        hidden = self._hidden_mask()
        last = 1 << (self.nlayers - 1)
        one, two = (int(code) >> 20) & hidden, (int(code) >> 8) & hidden
        if (int(code) & 0xff) != 1 or self.nlayers < 3 or one != (hidden & ~last) or not (two & last) or not self.tail_k_split:
            return None
        return torch.empty(int(_lib.load().nphm_mlp_eval_workspace_bytes()), dtype=torch.uint8, device=device)

    def _eval_points_raw(self, packed, state, xyz, add_input, code):
        lib = _lib.load()
        B, N, _ = xyz.shape
        out = torch.empty(B, N, self.n_out, dtype=torch.float32, device=xyz.device)
        stream = torch.cuda.current_stream(xyz.device).cuda_stream
        ws = self.eval_workspace(code, xyz.device)
        _lib.check(lib.nphm_mlp_eval_points_ws(*self._arch(), packed.data_ptr(), state.data_ptr(), xyz.data_ptr(),
                                               B, N, int(bool(add_input)), int(code), out.data_ptr(),
                                               ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0, stream),
                   "nphm_mlp_eval_points")
        return out

    def calibrate_two_pass(self, packed, state, sample_xyz, err_of=None, target=None):
        """Which hidden layers may run the two-term product xh wh + xl wh (weights rounded to the half format) on THIS
        checkpoint: the largest set whose output stays within ``numerics_target`` of the three-term product on
        ``sample_xyz`` [1,n,3] with the conditioning in ``state`` (row 0).  All layers at once if that holds; otherwise
        the layers are added in the order of their individual errors while the measured error of the set stays inside.
        Synchronises (one scalar per candidate); ~2 (best case) .. 2 nlayers small launches.  Returns (mask, report).
        ``err_of(mask) -> float`` / ``target``: another error measure and its bound (the fitting launches: value AND Jacobian
        on every conditioning row, _fit_err)."""
        fmt = self._format_code()
        if err_of is None:
            ref = self._eval_points_raw(packed, state, sample_xyz, False, fmt)
            err_of = lambda m: float((self._eval_points_raw(packed, state, sample_xyz, False, fmt | (m << 8)) - ref).abs().max())
        raw_err = err_of
        # a NaN / inf error (a non-finite sample point, an overflowing layer) must FAIL every comparison below: `nan > tgt` and
        # `nan <= tgt` are both false, which used to accept the layer
        err_of = lambda m: (lambda e: e if math.isfinite(e) else float("inf"))(raw_err(m))
        tgt = self.numerics_target if target is None else float(target)
        full = self._hidden_mask()
        e_all = err_of(full)
        report = {"target": tgt, "all_layers_err": e_all, "sample_points": int(sample_xyz.shape[1])}
        if e_all <= tgt:
            report.update(mask=full, err=e_all)
            return full, report
        layers = [l for l in range(1, self.nlayers) if (full >> l) & 1]
        single = sorted((err_of(1 << l), l) for l in layers)
        report["per_layer_err"] = {l: e for e, l in single}
        mask, err = 0, 0.0
        for e, l in single:
            if e > tgt:
                break
            trial = mask | (1 << l)
            et = err_of(trial)
            if et > tgt:
                break
            mask, err = trial, et
        report.update(mask=mask, err=err)
        return mask, report

    def _single_ok(self) -> bool:
        return self.allow_single_term and self.precision == "f16x3" and self.nlayers >= 2

    def _code(self, two_mask: int, one_mask: int = 0) -> int:
        """`numerics` argument (include/nphm_amd.h): format byte | two-term layer mask << 8 | single-term layer mask << 20"""
        hid = self._hidden_mask()
        one_mask &= hid
        return self._format_code() | ((two_mask & hid & ~one_mask) << 8) | (one_mask << 20)

    def calibrate_numerics(self, packed, state, sample_xyz):
        """The cheapest per-layer tiers of the plain evaluation that stay within ``numerics_target`` of the three-term product
        on ``sample_xyz``: -> (numerics code, report).  Order: the single-term product rn(x) wh in EVERY hidden layer (half
        the MFMAs of the two-term tier and, with twice the points per workgroup, half its weight bytes per point); that with the
        last hidden layer two-term (same workgroup shape); else the
        two-term layers of ``calibrate_two_pass`` and, of those, single-term layers added in the order of their individual
        errors while the measured error of the whole setting stays inside."""
        fmt = self._format_code()
        hid = self._hidden_mask()
        if not self._single_ok():
            mask, report = self.calibrate_two_pass(packed, state, sample_xyz)
            report.update(single_mask=0, single_term=False)
            return self._code(mask), report
        ref = self._eval_points_raw(packed, state, sample_xyz, False, fmt)
        _e = lambda two, one: float((self._eval_points_raw(packed, state, sample_xyz, False, self._code(two, one)) - ref).abs().max())
        err_of = lambda two, one: (lambda e: e if math.isfinite(e) else float("inf"))(_e(two, one))     # (NaN fails every comparison below)
        e_all = err_of(0, hid)
        if e_all <= self.numerics_target:
            return self._code(0, hid), {"target": self.numerics_target, "single_term": True, "single_mask": hid, "mask": 0,
                                        "err": e_all, "sample_points": int(sample_xyz.shape[1])}
        if self.nlayers >= 3:
            # ... but the LAST hidden layer two-term: still twice the points per workgroup (mlp_kernel.hip, TAIL2 - that layer runs
            # in two point halves, its weights are streamed twice, every other layer's once)
            tail = 1 << (self.nlayers - 1)
            e_tail = err_of(tail, hid & ~tail)
            if e_tail <= self.numerics_target:
                return self._code(tail, hid & ~tail), {"target": self.numerics_target, "single_term": False, "tail_two_term": True,
                                                       "single_mask": hid & ~tail, "mask": tail, "err": e_tail, "all_single_err": e_all,
                                                       "sample_points": int(sample_xyz.shape[1])}
        mask, report = self.calibrate_two_pass(packed, state, sample_xyz)
        report["all_single_err"] = e_all
        layers = [l for l in range(1, self.nlayers) if (mask >> l) & 1]
        per_layer = sorted((err_of(mask, 1 << l), l) for l in layers)
        report["per_layer_single_err"] = {l: e for e, l in per_layer}
        one, err = 0, report.get("err", 0.0)
        for e, l in per_layer:
            if e > self.numerics_target:
                break
            et = err_of(mask, one | (1 << l))
            if et > self.numerics_target:
                continue
            one, err = one | (1 << l), et
        report.update(single_mask=one, single_term=False, err=err)
        return self._code(mask, one), report

    def _numerics_code(self, packed, state, n_points, sample_fn):
        """`numerics` argument of this evaluation.  ``sample_fn()`` -> [1,n,3] points of THIS call (a strided subsample)."""
        fmt = self._format_code()
        if self.numerics == "fixed":
            if self.single_mask and self.precision != "f16x3":
                raise ValueError("DeepSDF.single_mask needs precision 'f16x3'")
            return self._code(int(self.two_pass_mask), int(self.single_mask))
        if self.numerics != "auto":
            raise ValueError(f"DeepSDF.numerics must be 'auto' or 'fixed', got {self.numerics!r}")
        if n_points < self.two_pass_min_points or torch.cuda.is_current_stream_capturing():
            return fmt                       # small or captured evaluations: the three-term product everywhere
        ws, bs = self._lin_params()
        key = tuple((t.data_ptr(), t._version) for t in ws + bs) + (self.precision, float(self.numerics_target), self._single_ok())
        sample = sample_fn()
        if self._two_pass_cache is None or self._two_pass_cache[0] != key:
            code, report = self.calibrate_numerics(packed, state, sample)
            self._two_pass_cache = (key, code, report)
            self._numerics_serial = getattr(self, "_numerics_serial", 0) + 1      # (reconstruction.shared_mlp_code)
            self.last_numerics = dict(report, precision=self.precision, verified_err=report.get("err", 0.0), calibrated_here=True)
            return code
        code = self._two_pass_cache[1]
        if code == fmt:
            return fmt
        # a later conditioning / point set inherits the calibrated tier only after it is VERIFIED on a sample of this call
        ref = self._eval_points_raw(packed, state, sample, False, fmt)
        err = float((self._eval_points_raw(packed, state, sample, False, code) - ref).abs().max())
        self.last_numerics = dict(self._two_pass_cache[2], precision=self.precision, verified_err=err, calibrated_here=False)
        if err > self.numerics_target:
            # this conditioning needs a more careful tier; the cache keeps the tightened one (every later call would
            # otherwise repeat verify -> fail -> recalibrate, ~2 nlayers launches and host syncs each)
            code, report = self.calibrate_numerics(packed, state, sample)
            self._two_pass_cache = (key, code, dict(report, tightened_for_conditioning=True))
            self._numerics_serial = getattr(self, "_numerics_serial", 0) + 1
            self.last_numerics = dict(report, precision=self.precision, verified_err=report.get("err", 0.0), calibrated_here=True,
                                      recalibrated_for_conditioning=True)
        return code

    def _jvp_split(self, R, n, device, align):
        """How a value+Jacobian launch over R rows x n points is cut: [(point_base, point_count, columns)].  Its workgroups
        hold 16 points (64 columns: value + three tangents); when they would fill between 1 and 1.5 rounds of the chip (the
        fitting loop: 5 x 1000 points = 315 workgroups on 256 CUs, the second round a fifth full) the first round takes as
        many whole rows-of-16 as fit and the REST runs as 8-point workgroups (32 columns, half the LDS: two per CU), whose
        round is shorter.  ``align``: granularity of the cut (16; 64 for the sigma'-saving form)."""
        if self.hidden_dim > 512 or os.environ.get("NPHM_AMD_JVP_SPLIT", "1") in ("0", ""):
            return [(0, 0, 64)]
        cus = torch.cuda.get_device_properties(device).multi_processor_count
        wgs = R * ((n + 15) // 16)
        if not (cus < wgs <= cus + cus // 2):
            return [(0, 0, 64)]
        n_a = ((cus // R) * 16) // align * align
        if n_a <= 0 or n_a >= n:
            return [(0, 0, 64)]
        # (the SHORT round first: whatever runs beside these launches on another stream - the fitting step's identity field - finds
        # free CUs at once and has left them again when the chip-filling round arrives; same result either way)
        if os.environ.get("NPHM_AMD_JVP_SMALL_FIRST", "1") not in ("0", ""):
            return [(n_a, n - n_a, 32), (0, n_a, 64)]
        return [(0, n_a, 64), (n_a, n - n_a, 32)]

    def _eval_jvp_raw(self, packed, state, xyz, code):
        lib = _lib.load()
        B, N, _ = xyz.shape
        out = torch.empty(B, N, 4, self.n_out, dtype=torch.float32, device=xyz.device)
        stream = torch.cuda.current_stream(xyz.device).cuda_stream
        _lib.check(lib.nphm_mlp_eval_points_jvp(*self._arch(), packed.data_ptr(), state.data_ptr(), xyz.data_ptr(), B, N, 0,
                                                out.data_ptr(), int(code), 0, 0, 64, None, stream), "nphm_mlp_eval_points_jvp")
        return out

    def _fit_err(self, packed, state, sample):
        """-> err_of(mask): deviation of the value + Jacobian launch with the two-term layers of ``mask`` from its three-term
        form on ``sample`` [B,n,3] (every conditioning row of ``state``), in units of the bounds: max(|d value| / fit_target,
        |d Jacobian| / fit_jacobian_target).  The fitting loop differentiates through these launches (Broyden's start
        Jacobian, the implicit-function gradient, fitting.py:99-106): the tangents are part of the criterion."""
        ref = self._eval_jvp_raw(packed, state, sample, 1)

        def err_of(mask):
            d = (self._eval_jvp_raw(packed, state, sample, 1 | (mask << 8)) - ref).abs()
            return max(float(d[:, :, 0].max()) / self.fit_target, float(d[:, :, 1:].max()) / self.fit_jacobian_target)
        return err_of

    @staticmethod
    def _fit_sample(xyz):
        n = xyz.shape[1]
        per_row = max(256, 4096 // max(1, xyz.shape[0]))
        s = xyz[:, :: max(1, n // per_row)][:, :per_row].contiguous().float()
        # (after a capture the points are the correspondence search's roots, diverged Broyden points included: a non-finite or
        # far-out point says nothing about the tiers - it is replaced by the origin)
        ok = torch.isfinite(s).all(dim=-1, keepdim=True) & (s.abs().amax(dim=-1, keepdim=True) < 10.0)
        return torch.where(ok, s, torch.zeros_like(s))

    def _fit_code(self, packed, state, xyz):
        """`numerics` argument of the tangent / Broyden / saving launches (``fit_numerics``).  xyz [B,N,3]: this call's points.
        "auto": split-f16 operands with the two-term layers of a mask calibrated per weight version on a sample of the first
        such call's points under ALL of its conditioning rows, value and Jacobian both (_fit_err); re-measured on the
        conditioning of the day by ``reverify_fit`` (the fitting loop calls it every ``fit_verify_every`` steps, outside the
        replayed graph, and re-captures when the mask shrank)."""
        if self.fit_numerics not in ("auto", "bf16x3", "f16x3"):
            raise ValueError(f"DeepSDF.fit_numerics must be 'auto', 'f16x3' or 'bf16x3', got {self.fit_numerics!r}")
        if self.hidden_dim > 512 or self.fit_numerics == "bf16x3":
            return 0                          # (the 1024-wide variant has bf16 tangent kernels only)
        if self.fit_numerics == "f16x3":
            return 1
        ws, bs = self._lin_params()
        key = tuple((t.data_ptr(), t._version) for t in ws + bs) + (float(self.fit_target), float(self.fit_jacobian_target))
        c = self._fit_cache
        self._fit_last = (packed, state, xyz)          # what reverify_fit measures on (inside a capture: the static tensors)
        if c is None or c[0] != key:
            if torch.cuda.is_current_stream_capturing() or xyz.shape[0] * xyz.shape[1] < 1024:
                return 1                      # nothing measured yet for these weights: three terms (split-f16)
            sample = self._fit_sample(xyz)
            mask, report = self.calibrate_two_pass(packed, state, sample, err_of=self._fit_err(packed, state, sample), target=1.0)
            report.update(value_target=self.fit_target, jacobian_target=self.fit_jacobian_target, rows=int(xyz.shape[0]))
            c = (key, mask, report)
            self._fit_cache = c
            self._fit_calls = 0
        elif c[1] and not torch.cuda.is_current_stream_capturing():
            # eager loops: the same re-measurement the graphed loop triggers (a fitting step issues ~6 of these launches)
            self._fit_calls = getattr(self, "_fit_calls", 0) + 1
            if self._fit_calls % (6 * max(1, int(self.fit_verify_every))) == 0 and xyz.shape[0] * xyz.shape[1] >= 1024:
                self.reverify_fit()
                c = self._fit_cache
        return 1 | (c[1] << 8)

    def reverify_fit(self) -> bool:
        """Measure the cached fitting mask on the most recent fitting launch's points and CURRENT conditioning rows (outside
        any capture); if it no longer holds, re-calibrate there and keep the intersection.  -> True if the mask changed (a
        captured step that baked it in must be recorded again)."""
        c, last = self._fit_cache, getattr(self, "_fit_last", None)
        if c is None or last is None or c[1] == 0 or self.fit_numerics != "auto" or torch.cuda.is_current_stream_capturing():
            return False
        packed, state, xyz = last
        sample = self._fit_sample(xyz)
        err_of = self._fit_err(packed, state, sample)
        e = err_of(c[1])
        c[2]["reverified_err"] = e
        if e <= 1.0:                              # (a NaN fails this test: the mask is measured again below)
            return False
        mask, report = self.calibrate_two_pass(packed, state, sample, err_of=err_of, target=1.0)
        mask &= c[1]
        report.update(value_target=self.fit_target, jacobian_target=self.fit_jacobian_target, tightened_from=c[1], mask=mask)
        self._fit_cache = (c[0], mask, report)
        return mask != c[1]                       # only a CHANGED mask makes a recorded step stale

    def forward_hip(self, xyz, cond_rows, add_input=False):
        """xyz [B,N,3] fp32 on a ROCm device, cond_rows [B, lat_dim] -> [B,N,out_dim]
        (+ xyz on the first three outputs if ``add_input``)."""
        B, N, _ = xyz.shape
        packed, state = self.prepare_latent(cond_rows)
        xyz = xyz.contiguous().float()

        def sample():
            step = max(1, N // 4096)
            return xyz[:1, ::step][:, :4096].contiguous()

        code = self._numerics_code(packed, state, B * N, sample) if B == 1 else self._format_code()
        return self._eval_points_raw(packed, state, xyz, add_input, code)

    def forward_hip_jvp(self, xyz, cond_rows, add_input=False, inverse=False):
        """Value and spatial Jacobian in one fused launch (forward-mode tangents carried through the
        same GEMMs): xyz [B,N,3], cond_rows [B,lat_dim] -> [B,N,4,out_dim] with [:,:,0] = f(x)
        (+ x if ``add_input``) and [:,:,1+c,i] = d f_i / d x_c (+ identity if ``add_input``).  ``inverse``: -> (that, the
        inverse [B,N,3,3] of the Jacobian of the first three outputs - rows = outputs, columns = x, y, z) from the same launch."""
        lib = _lib.load()
        B, N, _ = xyz.shape
        packed, state = self.prepare_latent(cond_rows)
        xyz = xyz.contiguous().float()
        out = torch.empty(B, N, 4, self.n_out, dtype=torch.float32, device=xyz.device)
        jinv = torch.empty(B, N, 3, 3, dtype=torch.float32, device=xyz.device) if inverse else None
        stream = torch.cuda.current_stream(xyz.device).cuda_stream
        code = self._fit_code(packed, state, xyz)
        for p0, cnt, cols in self._jvp_split(B, N, xyz.device, 16):
            _lib.check(lib.nphm_mlp_eval_points_jvp(*self._arch(), packed.data_ptr(), state.data_ptr(), xyz.data_ptr(),
                                                    B, N, int(bool(add_input)), out.data_ptr(), code, p0, cnt, cols,
                                                    None if jinv is None else jinv.data_ptr(), stream),
                       "nphm_mlp_eval_points_jvp")
        return (out, jinv) if inverse else out

    def broyden_hip(self, obs, x_init, jinv_init, cond_rows, max_steps, cvg_thresh, dvg_thresh, eps=1e-6, posed_init=None):
        """Roots of x + f(x) = obs by Broyden's method, fused around the network in one launch
        (nphm_mlp_broyden).  obs / x_init [B,N,3], jinv_init [B,N,3,3], cond_rows [B,lat_dim] ->
        (x [B,N,3], smallest residual norm [B,N], converged [B,N] bool).  ``posed_init`` [B,N,3] (any point stride):
        x_init + f(x_init) when the caller holds it already - the first evaluation is then skipped."""
        lib = _lib.load()
        B, N, _ = x_init.shape
        packed, state = self.prepare_latent(cond_rows)
        dev = x_init.device
        obs, x_init, jinv_init = obs.contiguous().float(), x_init.contiguous().float(), jinv_init.contiguous().float()
        x = torch.empty(B, N, 3, dtype=torch.float32, device=dev)
        diff = torch.empty(B, N, dtype=torch.float32, device=dev)
        valid = torch.empty(B, N, dtype=torch.uint8, device=dev)
        stream = torch.cuda.current_stream(dev).cuda_stream
        code = self._fit_code(packed, state, x_init)
        stride = None
        if posed_init is not None and posed_init.dtype == torch.float32 and posed_init.shape == x_init.shape and posed_init.stride(-1) == 1:
            ps = posed_init.stride(1)
            if posed_init.stride(0) == ps * N:                # the rows collapse into one point stride
                stride = ps
        if stride is not None:
            _lib.check(lib.nphm_mlp_broyden_from(*self._arch(), packed.data_ptr(), state.data_ptr(), obs.data_ptr(),
                                                 x_init.data_ptr(), jinv_init.data_ptr(), posed_init.data_ptr(), stride, B, N,
                                                 int(max_steps), float(cvg_thresh), float(dvg_thresh), float(eps), x.data_ptr(),
                                                 diff.data_ptr(), valid.data_ptr(), code, stream), "nphm_mlp_broyden_from")
        else:
            _lib.check(lib.nphm_mlp_broyden(*self._arch(), packed.data_ptr(), state.data_ptr(), obs.data_ptr(),
                                            x_init.data_ptr(), jinv_init.data_ptr(), B, N, int(max_steps),
                                            float(cvg_thresh), float(dvg_thresh), float(eps), x.data_ptr(),
                                            diff.data_ptr(), valid.data_ptr(), code, stream), "nphm_mlp_broyden")
        return x, diff, valid.view(torch.bool)           # the kernel writes 0 / 1 bytes

    def _hip_rows(self, xyz, cond, cond_grad_ok=False):
        """How the HIP tier can serve this call: returns (xyz_view [R,n,3], cond_rows [R,lat_dim]) or
        None (-> composite tier).  Raises on a CPU tensor without the explicit opt-in.  ``cond_grad_ok``: the
        caller can differentiate with respect to the conditioning (``forward_hip_cond_grad``), so a graph that
        only needs THAT gradient (frozen parameters, detached points: the fitting loop) stays on the HIP tier.

        Besides a row-constant conditioning ([B,1,L] or a ``repeat`` along the points) it recognises
        the flattened batch the reference's root finder passes (iterative_root_finding.py:137-139):
        xyz [1, S*n, 3] with a conditioning that is constant on S equal segments, which is re-viewed
        as S batch rows."""
        if self.backend == "composite":
            return None
        if not xyz.is_cuda:
            raise _lib.NphmAmdError(
                "DeepSDF: tensors are on the CPU; the HIP path needs a ROCm device "
                "(set module.backend = 'composite' explicitly for the PyTorch formulation)")
        needs_graph = torch.is_grad_enabled() and (
            xyz.requires_grad or cond.requires_grad or any(p.requires_grad for p in self.parameters()))
        if needs_graph:
            cond_only = (cond_grad_ok and not xyz.requires_grad and not any(p.requires_grad for p in self.parameters())
                         and cond.shape[1] == 1 and self.hip_backward_supported())
            if not cond_only:
                return None
        if xyz.dtype != torch.float32 or not self.hip_supported():
            return None
        B, N = xyz.shape[0], xyz.shape[1]
        if cond.shape[1] == 1:
            return xyz, cond.reshape(cond.shape[0], cond.shape[2])         # (a view: the backward of a select costs two launches)
        if cond.shape[1] != N:
            return None
        change = (cond[:, 1:] != cond[:, :-1]).any(dim=-1)                 # [B, N-1]
        if B > 1:
            return (xyz, cond[:, 0, :]) if not bool(change.any()) else None
        edges = change[0].nonzero().flatten()                             # one host sync
        if edges.numel() == 0:
            return xyz, cond[:, 0, :]
        if edges.numel() > 64:                                            # per-point conditioning
            return None
        # segment length = gcd of the run boundaries (runs may merge when neighbouring segments
        # carry the same code, e.g. an observation sampled twice in a fitting batch)
        seg = N
        for e in (edges + 1).tolist():
            seg = math.gcd(seg, int(e))
        if seg < 64:
            return None
        return xyz.reshape(N // seg, seg, 3), cond[0, ::seg, :]

    def forward(self, xyz, lat_rep, anchors=None):
        squeeze = xyz.dim() < 3
        x3 = xyz.unsqueeze(0) if squeeze else xyz
        plan = self._hip_rows(x3, lat_rep, cond_grad_ok=True)
        if plan is not None:
            fwd = self.forward_hip_cond_grad if (torch.is_grad_enabled() and lat_rep.requires_grad) else self.forward_hip
            out = fwd(*plan).reshape(x3.shape[0], x3.shape[1], self.n_out)
            return (out.squeeze(0) if squeeze else out), None
        if lat_rep.dim() == 3 and self.train_tier_serves(x3, lat_rep):
            out = self.evaluate_train_hip(self._embed(x3), lat_rep)
            return (out.squeeze(0) if squeeze else out), None
        return self.evaluate(self._embed(xyz), lat_rep, gemm_hip=lat_rep.dim() == 3 and self.gemm_tier_serves(x3, lat_rep)), None


class _CompressCondFn(torch.autograd.Function):
    """cond [B,1,32+e] = [compressor([z_id | anchors]) on every row | z_ex[b]] (deepSDF.py:212-223 for ONE identity on every
    row: the fitting loops) in one launch, and one launch back (``nphm_compress_condition`` / ``_backward``) - a cat, a fused
    head launch and a cat forward, a sum over the rows and the head's backward launch in the composite formulation.  The
    gradient of z_ex is a column slice of the incoming gradient (a view)."""

    @staticmethod
    def forward(ctx, z_id, anchors1, z_ex, weight, bias):
        lib = _lib.load()
        B, E, O = z_ex.shape[0], z_ex.shape[-1], weight.shape[0]
        cond = torch.empty(B, 1, O + E, dtype=torch.float32, device=z_ex.device)
        w, b = weight.detach().contiguous(), bias.detach().contiguous()
        _lib.check(lib.nphm_compress_condition(w.data_ptr(), b.data_ptr(), z_id.detach().data_ptr(), z_id.numel(), anchors1.detach().data_ptr(),
                                               anchors1.numel(), O, z_ex.detach().data_ptr(), B, E, cond.data_ptr(),
                                               torch.cuda.current_stream(z_ex.device).cuda_stream), "nphm_compress_condition")
        ctx.save_for_backward(w, b)
        ctx.meta = (z_id.shape, anchors1.shape, B, E, O)
        return cond

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_cond):
        lib = _lib.load()
        w, b = ctx.saved_tensors
        s_id, s_anc, B, E, O = ctx.meta
        g = g_cond.contiguous().float()
        g_id = torch.empty(s_id, dtype=torch.float32, device=g.device)
        g_anc = torch.empty(s_anc, dtype=torch.float32, device=g.device)
        _lib.check(lib.nphm_compress_condition_backward(w.data_ptr(), b.data_ptr(), g_id.numel(), g_anc.numel(), O, g.data_ptr(), B, E,
                                                        g_id.data_ptr(), g_anc.data_ptr(), torch.cuda.current_stream(g.device).cuda_stream),
                   "nphm_compress_condition_backward")
        return g_id, g_anc, g[..., O:], None, None


class DeformationNetwork(nn.Module):
    """Forward deformation field F_ex (deepSDF.py:118-239).  Conditioning modes: 'glob_only',
    'expr_only', 'interpolate', 'compress' (the NPHM one: identity code + anchors are projected to
    32 dims from ROW 0 of the latent and concatenated with the expression code), 'GNN'."""

    def __init__(self, mode, lat_dim_expr, lat_dim_id, lat_dim_glob_shape, lat_dim_loc_shape, n_loc,
                 anchors, hidden_dim, nlayers=8, out_dim=1, input_dim=3):
        super().__init__()
        self.mode = mode
        self.lat_dim_glob_shape = lat_dim_glob_shape
        self.lat_dim_loc_shape = lat_dim_loc_shape
        self.lat_dim_expr = lat_dim_expr
        self.input_dim = input_dim
        self.num_kps = n_loc
        self.out_dim = out_dim + 1

        if mode == "glob_only":
            self.lat_dim = lat_dim_glob_shape + lat_dim_expr
        elif mode == "expr_only":
            self.lat_dim = lat_dim_expr
        elif mode == "interpolate":
            self.lat_dim = lat_dim_glob_shape + lat_dim_expr + lat_dim_loc_shape
        elif mode == "compress":
            self.lat_dim = lat_dim_expr + lat_dim_id
            self.compressor = nn.Sequential(
                nn.Linear((lat_dim_loc_shape + 3) * n_loc + lat_dim_loc_shape + lat_dim_glob_shape, 32))
        elif mode == "GNN":
            self.lat_dim = lat_dim_expr * 2
            self.pos_enc = nn.Sequential(nn.Linear(3, lat_dim_loc_shape), nn.ReLU(),
                                         nn.Linear(lat_dim_loc_shape, lat_dim_loc_shape))
            self.local_combiner = nn.Sequential(nn.Linear(lat_dim_loc_shape, lat_dim_loc_shape), nn.ReLU(),
                                                nn.Linear(lat_dim_loc_shape, lat_dim_loc_shape))
            self.global_combiner = nn.Sequential(
                nn.Linear(lat_dim_glob_shape + n_loc * lat_dim_loc_shape, 512), nn.ReLU(),
                nn.Linear(512, lat_dim_expr))
        else:
            raise ValueError("Unknown mode!")

        print("creating DeepSDF with...")
        print("lat dim", self.lat_dim)
        print("hidden_dim", hidden_dim)
        self.defDeepSDF = DeepSDF(lat_dim=self.lat_dim, hidden_dim=hidden_dim, nlayers=nlayers,
                                  geometric_init=False, out_dim=out_dim, input_dim=input_dim).float()
        self.anchors = anchors

    @contextmanager
    def condition_scope(self):
        """Inside the scope, calls that pass the SAME ``lat_rep`` / ``anchors`` tensors (same storage and version;
        no gradient involved) share one conditioning row and one kernel prologue - the fitting step evaluates the
        field four times per step on one set of codes (search Jacobian, Broyden, posed points, Jacobian of the
        implicit differentiation).  The scope holds the tensors, so an address cannot be recycled under it."""
        self._cond_scope, self.defDeepSDF._state_scope = {}, {}
        try:
            yield self
        finally:
            self._cond_scope, self.defDeepSDF._state_scope = None, None

    def _condition(self, xyz, lat_rep, anchors):
        """Conditioning vector [B,Lr,lat_dim] (Lr = 1 when it is constant along the points)."""
        scope = getattr(self, "_cond_scope", None)
        key = None
        wants_graph = torch.is_grad_enabled() and (lat_rep.requires_grad or (anchors is not None and anchors.requires_grad))
        if scope is not None and self.mode == "compress" and not self.training and anchors is not None:
            # (a detached alias has the address, version, shape and strides of its source: same key)
            key = (lat_rep.data_ptr(), lat_rep._version, tuple(lat_rep.shape), tuple(lat_rep.stride()),
                   anchors.data_ptr(), anchors._version, tuple(anchors.shape), tuple(anchors.stride()))
            hit = scope.get(key)
            if hit is not None and (hit[3] or not wants_graph):
                return hit[0] if wants_graph else hit[0].detach()
        cond = self._condition_impl(xyz, lat_rep, anchors)
        if key is not None:
            scope[key] = (cond, lat_rep, anchors, cond.requires_grad)
        return cond

    def prime_condition(self, lat_rep, anchors, parts=None):
        """Inside a ``condition_scope``: evaluate the conditioning of (lat_rep, anchors) ONCE, with its autograd graph, so that
        the step's later calls - the no-grad ones of the correspondence search and the differentiable one at the roots -
        share it (a fitting step otherwise runs the compressor twice).  No-op outside a scope / for other modes.

        ``parts`` = (z_id [1,1,L_id], z_ex [B,1,e], anchors [1,K,3]) states that ``lat_rep`` is [z_id on every row | z_ex] and
        ``anchors`` that one set on every row (the fitting loops: one identity, B sampled observations): the compressor then
        runs on ONE row and the gradients reach z_id / the anchors without an expand-and-sum over the rows.  Same values."""
        if getattr(self, "_cond_scope", None) is None or self.mode != "compress" or self.training or anchors is None:
            return
        if parts is not None and not (parts[0].shape[0] == 1 and parts[2].shape[0] == 1 and parts[1].shape[0] == lat_rep.shape[0]):
            parts = None                          # not "one identity on every row": the generic evaluation
        if parts is None:
            self._condition(lat_rep[:, :1, :3], lat_rep, anchors)
            return
        z_id, z_ex, anchors1 = parts
        from .ensembled_deepsdf import frozen_head
        lin = self.compressor[0]
        if (len(self.compressor) == 1 and z_id.is_cuda and os.environ.get("NPHM_AMD_FIT_FUSED", "1") not in ("0", "")
                and not any(p.requires_grad for p in lin.parameters()) and lin.bias is not None and lin.in_features <= 1536
                and all(t.dtype == torch.float32 and t.is_contiguous() for t in (z_id, z_ex, anchors1))
                and z_id.numel() + anchors1.numel() == lin.in_features and z_ex.dim() == 3 and z_ex.shape[1] == 1):
            cond = _CompressCondFn.apply(z_id, anchors1, z_ex, lin.weight, lin.bias)     # [B,1,32+e]: one launch each way
        else:
            packed = torch.cat([z_id.reshape(1, -1), anchors1.reshape(1, -1)], dim=-1)
            comp = frozen_head(self.compressor, packed, False)                       # [1,32]
            cond = torch.cat([comp.unsqueeze(1).expand(z_ex.shape[0], 1, -1), z_ex], dim=-1)
        key = (lat_rep.data_ptr(), lat_rep._version, tuple(lat_rep.shape), tuple(lat_rep.stride()),
               anchors.data_ptr(), anchors._version, tuple(anchors.shape), tuple(anchors.stride()))
        self._cond_scope[key] = (cond, lat_rep, anchors, cond.requires_grad)

    def _condition_impl(self, xyz, lat_rep, anchors):
        B, N, _ = xyz.shape
        e = self.lat_dim_expr
        g = self.lat_dim_glob_shape
        if self.mode == "glob_only":
            return torch.cat([lat_rep[..., :g], lat_rep[..., -e:]], dim=-1)
        if self.mode == "expr_only":
            return lat_rep[..., -e:]
        if self.mode == "interpolate":
            loc = lat_rep[:, 0, g:-e - self.lat_dim_loc_shape].view(B, self.num_kps, self.lat_dim_loc_shape)
            interp = sample_point_feature(xyz[..., :3], anchors[:, 0, :, :3], loc.unsqueeze(1), background=False)
            Lr = lat_rep.shape[1]
            head = lat_rep[..., :g] if Lr == N else lat_rep[..., :g].expand(B, N, g)
            tail = lat_rep[..., -e:] if Lr == N else lat_rep[..., -e:].expand(B, N, e)
            return torch.cat([head, interp, tail], dim=-1)
        if self.mode == "compress":
            a0 = anchors[:, 0] if anchors.dim() == 4 else anchors              # row 0 only
            packed = torch.cat([lat_rep[:, 0, :-e], a0.reshape(B, -1)], dim=-1)
            from .ensembled_deepsdf import frozen_head
            comp = frozen_head(self.compressor, packed, False).unsqueeze(1)     # [B,1,32]; one launch when the weights are frozen
            if self.training:
                comp = comp + torch.randn(B, N, comp.shape[-1], device=comp.device) / 200
            Lr = max(comp.shape[1], lat_rep.shape[1])
            return torch.cat([comp.expand(B, Lr, -1), lat_rep[..., -e:].expand(B, Lr, e)], dim=-1)
        if self.mode == "GNN":
            pos = self.pos_enc(anchors[:, 0, :, :])
            loc = lat_rep[:, 0, g:g + self.num_kps * self.lat_dim_loc_shape].view(B, self.num_kps, 32)
            loc = self.local_combiner(pos + loc)
            comb = self.global_combiner(torch.cat([lat_rep[:, 0, :g], loc.view(B, -1)], dim=-1)).unsqueeze(1)
            Lr = lat_rep.shape[1]
            return torch.cat([comb.expand(B, Lr, -1), lat_rep[..., -e:]], dim=-1)
        raise ValueError("Unknown mode")

    def forward(self, xyz: torch.Tensor, lat_rep: torch.Tensor, anchors: Optional[torch.Tensor]):
        """xyz [B,N,3]; lat_rep [B,N or 1,·] = [z_id | z_ex]; anchors [B,N,K,3] or [B,K,3].
        Returns (offsets pred[..., :3], remaining features pred[..., -1:])."""
        if xyz.dim() < 3:
            xyz = xyz.unsqueeze(0)
        cond = self._condition(xyz, lat_rep, anchors)
        # the compressor / latent slices stay ordinary autograd; the backbone is differentiated by the HIP backward
        # kernel when only the conditioning needs a gradient (compressor parameters frozen like the backbone's)
        own_frozen = not any(p.requires_grad for p in self.parameters())
        plan = self.defDeepSDF._hip_rows(xyz, cond, cond_grad_ok=own_frozen)
        if plan is not None:
            fwd = (self.defDeepSDF.forward_hip_cond_grad if (torch.is_grad_enabled() and cond.requires_grad)
                   else self.defDeepSDF.forward_hip)
            pred = fwd(*plan).reshape(xyz.shape[0], xyz.shape[1], -1)
        elif self.defDeepSDF.train_tier_serves(xyz, cond):
            pred = self.defDeepSDF.evaluate_train_hip(self.defDeepSDF._embed(xyz), cond)     # trainable backbone: the dense training tier
        else:
            pred = self.defDeepSDF.evaluate(self.defDeepSDF._embed(xyz), cond, gemm_hip=self.defDeepSDF.gemm_tier_serves(xyz, cond))
        return pred[..., :3], pred[..., -1:]

    @property
    def backend(self):
        return self.defDeepSDF.backend

    @backend.setter
    def backend(self, value):
        self.defDeepSDF.backend = value

    def jacobian(self, xyz, lat_rep, anchors, inverse=False):
        """Posed points x + F_ex(x) [B,N,3] and the Jacobian d (x + F_ex) / d x [B,N,3,3]
        ([..., i, c] = d posed_i / d x_c — the layout of diff_operators.jac) in ONE fused launch
        instead of one forward + three autograd VJPs.  Detached results; returns None when the HIP
        tier cannot serve the call (CPU / composite backend / per-point conditioning / training-mode
        noise), so callers fall back to autograd."""
        if xyz.dim() < 3:
            xyz = xyz.unsqueeze(0)
        if self.backend == "composite" or not xyz.is_cuda or self.defDeepSDF.n_out < 3:
            return None
        with torch.no_grad():
            x = xyz.detach()
            cond = self._condition(x, lat_rep.detach(), None if anchors is None else anchors.detach())
            plan = self.defDeepSDF._hip_rows(x, cond)
            if plan is None:
                return None
            out = self.defDeepSDF.forward_hip_jvp(*plan, add_input=True, inverse=inverse)
            jinv = None
            if inverse:
                out, jinv = out
                jinv = jinv.reshape(x.shape[0], x.shape[1], 3, 3)
            out = out.reshape(x.shape[0], x.shape[1], 4, -1)
        if inverse:                        # (the inverse of the returned Jacobian, from the same launch)
            return out[:, :, 0, :3], out[:, :, 1:, :3].transpose(-1, -2), jinv
        return out[:, :, 0, :3], out[:, :, 1:, :3].transpose(-1, -2)

    def posed_and_jacobian(self, xyz, lat_rep, anchors, inverse=False):
        """(x + F_ex(x) [B,N,3] differentiable w.r.t. the conditioning, d (x + F_ex) / d x [B,N,3,3] detached) in ONE
        launch - ``forward`` + ``jacobian`` at the same points, as the fitting step needs them at the canonical
        correspondences (fitting.py:99-103).  None when the HIP autograd tier cannot serve the call (see ``forward``)."""
        if xyz.dim() < 3:
            xyz = xyz.unsqueeze(0)
        if self.backend == "composite" or not xyz.is_cuda or self.defDeepSDF.n_out < 3 or xyz.requires_grad:
            return None
        cond = self._condition(xyz, lat_rep, anchors)
        if not (torch.is_grad_enabled() and cond.requires_grad) or any(p.requires_grad for p in self.parameters()):
            return None
        plan = self.defDeepSDF._hip_rows(xyz, cond, cond_grad_ok=True)
        if plan is None:
            return None
        B, N = xyz.shape[0], xyz.shape[1]
        jinv = None
        if inverse:
            val, jac, jinv = _MlpCondFn.apply(self.defDeepSDF, plan[0], plan[1], True, True, True)
            jinv = jinv.reshape(B, N, 3, 3)
        else:
            val, jac = _MlpCondFn.apply(self.defDeepSDF, plan[0], plan[1], True, True)
        val, jac = val.reshape(B, N, -1), jac.reshape(B, N, 3, -1)
        if val.shape[-1] != 3:             # (a full-range slice would still cost a zero-fill + copy in the backward pass)
            val, jac = val[..., :3], jac[..., :3]
        if inverse:                        # (+ the inverse of that Jacobian, from the same launch)
            return val, jac.transpose(-1, -2).detach(), jinv
        return val, jac.transpose(-1, -2).detach()

    def implicit_root(self, roots, lat_rep, anchors):
        """x_c = roots - J^-1 (F(roots) - F(roots).detach()) with F = x + F_ex(x; z) (fitting.py:99-106): the detached roots
        of the correspondence search, made differentiable w.r.t. the conditioning by the implicit function theorem - value,
        Jacobian, its inverse and the state of the backward in ONE launch, and the -J^-T of the gradient inside the backward
        kernel.  [B,N,3], or None when the HIP autograd tier cannot serve the call (see ``posed_and_jacobian``)."""
        if roots.dim() < 3:
            roots = roots.unsqueeze(0)
        if self.backend == "composite" or not roots.is_cuda or self.defDeepSDF.n_out != 3 or roots.requires_grad:
            return None
        cond = self._condition(roots, lat_rep, anchors)
        if not (torch.is_grad_enabled() and cond.requires_grad) or any(p.requires_grad for p in self.parameters()):
            return None
        plan = self.defDeepSDF._hip_rows(roots, cond, cond_grad_ok=True)
        if plan is None:
            return None
        xc, _, _ = _MlpCondFn.apply(self.defDeepSDF, plan[0], plan[1], True, True, True, True)
        return xc.reshape(roots.shape)

    def broyden(self, obs, x_init, jinv_init, lat_rep, anchors, max_steps=15, cvg_thresh=1e-6, dvg_thresh=0.2,
                eps=1e-6, posed_init=None):
        """Canonical correspondences x_c with x_c + F_ex(x_c) = obs for all points in ONE fused launch
        (the reference iterates <= max_steps + 1 forwards with a host sync each,
        iterative_root_finding.py:5-71).  obs / x_init [B,N,3], jinv_init [B,N,3,3], lat_rep / anchors as
        for ``forward``.  Returns {'result' [B*N,3,1], 'diff' [B*N], 'valid_ids' [B*N]} like the
        reference's broyden, or None when the HIP tier cannot serve the call."""
        if self.backend == "composite" or not x_init.is_cuda or self.defDeepSDF.n_out < 3:
            return None
        with torch.no_grad():
            x0 = x_init.detach()
            cond = self._condition(x0, lat_rep.detach(), None if anchors is None else anchors.detach())
            plan = self.defDeepSDF._hip_rows(x0, cond)
            if plan is None:
                return None
            xv, rows = plan
            R, n = xv.shape[0], xv.shape[1]
            if posed_init is not None and tuple(posed_init.shape) != (R, n, 3):
                posed_init = None                              # (a re-viewed batch: let the kernel evaluate the start itself)
            x, diff, valid = self.defDeepSDF.broyden_hip(obs.detach().reshape(R, n, 3), xv,
                                                         jinv_init.detach().reshape(R, n, 3, 3), rows, max_steps,
                                                         cvg_thresh, dvg_thresh, eps, posed_init=posed_init)
        return {"result": x.reshape(-1, 3, 1), "diff": diff.reshape(-1), "valid_ids": valid.reshape(-1)}

    def canonical_points(self, xyz, lat_rep, anchors):
        """x + F_ex(x) in one fused launch (HIP tier) — the canonicalisation step of
        get_logits_backward / deform_mesh (models/reconstruction.py:44-46, :83-84)."""
        if xyz.dim() < 3:
            xyz = xyz.unsqueeze(0)
        cond = self._condition(xyz, lat_rep, anchors)
        plan = self.defDeepSDF._hip_rows(xyz, cond) if self.defDeepSDF.n_out >= 3 else None
        if plan is not None:
            out = self.defDeepSDF.forward_hip(*plan, add_input=True)
            return out.reshape(xyz.shape[0], xyz.shape[1], -1)[..., :3]
        pred = self.defDeepSDF.evaluate(self.defDeepSDF._embed(xyz), cond)
        return xyz[..., :3] + pred[..., :3]
