"""Operators of a training step around the decoders: the table of latent codes and its gradient, the dense layer in 16-bit storage
with its epilogue, the global gradient norm and clipping (what scripts/training/train.py does with nn.Embedding, nn.Linear and
clip_grad_norm_ between ``compute_loss`` and the optimisers, src/NPHM/models/training.py:111-135).

    codes = LatentCodes(n_subjects, 1344, max_norm=1.0, sparse=True, device="cuda")      # an nn.Embedding: same state_dict
    loss = weighted_total(compute_loss(batch, decoder, codes, device), lambdas)
    loss.backward()
    clip_grad_norm_(decoder.parameters(), 0.1)
    clip_grad_norm_(codes.parameters(), 0.1)                                            # row gradients too

Every function runs on libnphm_amd.so (csrc/rows_kernels.hip, clip_kernels.hip, layer16_kernels.hip; csrc/torch_ops.cpp checks its
arguments, allocates and holds its autograd node), on the current stream of its tensors' device.  It raises ``ValueError`` /
``TypeError`` for what it does not take and ``NphmAmdError`` if the library is missing or a call fails; there is no PyTorch fallback,
CPU tensors are refused, and so are forward-mode (dual) tensors, with ``NotImplementedError``.  Results are the same bits from run to run.  All of it can be captured into a graph, except where a
line says that it waits for the device.  (A backward pass is captured on leaves of which no graph of eager calls is alive: autograd would
make the default stream wait for the capture, which it cannot.  Where the operators' own gradients would go to such a leaf they raise.)"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from . import _lib

_ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "softplus": 4}
_CODES = {torch.float32, torch.bfloat16, torch.float16}


class _Ops:
    """The operators of libnphm_torch.so; the library is loaded at the first use of one."""

    def __getattr__(self, name):
        ops = _lib.load_torch()
        op = _lib.torch_clip if name == "clip" else getattr(ops, name).default

        def call(*args):
            try:
                return op(*args)
            except RuntimeError as e:
                msg = str(e)
                if msg.startswith("nphm: "):
                    raise _lib.NphmAmdError(msg.split("\n", 1)[0][6:]) from None
                if "Expected a value of type" in msg:
                    raise TypeError(msg.split("\n", 1)[0]) from None
                raise
        setattr(self, name, call)
        return call


_ops = _Ops()


# ---- rows of a table ---------------------------------------------------------------------------------------------------------

def lookup_rows(table, idx, scale=1.0, padding_idx=None, sparse=False):
    """scale * table[idx] for a table [V, D] (fp32, bf16 or fp16) and int32 / int64 indices of any shape: [*idx.shape, D] in the table's type,
    the product in fp32.  Differentiable (once) w.r.t. the table: a dense gradient (``lookup_rows_grad``) or, with ``sparse``, a
    sparse one with an entry for every index (``LatentCodes`` and ``clip_grad_norm_`` coalesce it where torch's optimisers cannot).  Row
    `padding_idx` is read like any other and gets no gradient.  An index outside the table gives a row of NaN and adds nothing to the
    gradient (nothing on the host looks at the indices)."""
    return _ops.lookup_rows(table, idx, scale, padding_idx, 1 if sparse else 0)


def lookup_rows_grad(grad, idx, num_rows, scale=1.0, padding_idx=None):
    """Gradient of ``lookup_rows`` w.r.t. its table of `num_rows` rows: [num_rows, D] of grad's type, ``scale`` times the sum of the rows
    of `grad` [*idx.shape, D] that name a row; zeros in rows that none names and in row `padding_idx`.  Sums are in fp32, in the
    order of the indices.  For programs that keep their own backward pass; autograd calls it by itself.  The result is part of no graph."""
    return _ops.lookup_rows_grad(grad, idx, num_rows, scale, padding_idx)


def renorm_rows_(table, idx, max_norm):
    """Rows of `table` that `idx` names and whose 2-norm is above `max_norm` are scaled down to it, in place, each once
    (nn.Embedding's max_norm, training.py:36-40)."""
    _ops.renorm_rows_(table, idx, max_norm)
    return table


# torch.sparse's coalesce, which torch.optim.SparseAdam calls, leaves the columns of wide rows as the memory was (PyTorch 2.10 on ROCm: of D
# columns the first 256 + 4 (ceil(D / 256) - 1) are written, found with rows of 64 to 2048).  It leaves a coalesced gradient alone.
_COALESCED_BY_TORCH = 256


def _needs_fold(g):
    """whether torch would coalesce the row gradient `g` on the device and lose columns"""
    v = g._values()
    return (v.is_cuda and v.dtype in _CODES and g.sparse_dim() == 1 and not g.is_coalesced() and v.shape[0] > 0
            and v[0].numel() > _COALESCED_BY_TORCH and not torch.cuda.is_current_stream_capturing())


@torch.no_grad()
def _folded(g):
    """The row gradient `g` coalesced: every row once, in ascending order, the sums in fp32 in the order of the entries (waits for the device)."""
    v = g._values()
    rows, place = torch.unique(g._indices()[0], return_inverse=True)
    sums = lookup_rows_grad(v.reshape(v.shape[0], -1), place, rows.numel()).view(rows.numel(), *v.shape[1:])
    return torch.sparse_coo_tensor(rows[None], sums, g.shape, is_coalesced=True, check_invariants=False)


def _fold_grad(p):
    if p.grad is not None and p.grad.is_sparse and _needs_fold(p.grad):
        p.grad = _folded(p.grad)


class LatentCodes(nn.Embedding):
    """The table of latent codes of the trainers (nn.Embedding(n, lat_dim, max_norm=1.0, sparse=True), training.py:36-40) on
    ``lookup_rows`` / ``renorm_rows_``; parameters, initialisation and state_dict are nn.Embedding's.  ``scale`` multiplies the looked-up
    rows.  With ``sparse``, codes of more than 256 entries get their ``weight.grad`` coalesced when a backward pass has left it (which waits for
    the device; not while a graph is captured): torch.optim.SparseAdam takes it as it is, where torch would lose columns of it.  Padding in
    a batch is an entry of zeros for its own row there: no optimiser moves a row by it.
    ``backend = "composite"`` computes the same with torch's embedding (CPU tensors need it, as in the decoders, and so do ``norm_type`` other than
    2 and ``scale_grad_by_freq``)."""

    def __init__(self, num_embeddings, embedding_dim, padding_idx=None, max_norm=None, scale=1.0, sparse=False, device=None, dtype=None,
                 norm_type=2.0, scale_grad_by_freq=False, _weight=None, _freeze=False):
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx, max_norm=max_norm, norm_type=norm_type,
                         scale_grad_by_freq=scale_grad_by_freq, sparse=sparse, _weight=_weight, _freeze=_freeze, device=device, dtype=dtype)
        if not math.isfinite(scale):
            raise ValueError(f"LatentCodes: scale {scale}")
        self.scale = float(scale)
        self.backend = "hip"            # "hip" | "composite"

    def forward(self, idx):
        w = self.weight
        if self.sparse and w.is_cuda and w.is_leaf and w.requires_grad and w.shape[1] > _COALESCED_BY_TORCH:
            # (looked for in every call: a copied or unpickled module's weight has no hooks)
            if _fold_grad not in (w._post_accumulate_grad_hooks or {}).values():
                w.register_post_accumulate_grad_hook(_fold_grad)
        if self.backend == "composite":
            rows = super().forward(idx)
            return rows if self.scale == 1.0 else rows * self.scale
        if self.scale_grad_by_freq or (self.max_norm is not None and self.norm_type != 2):
            raise ValueError("LatentCodes: scale_grad_by_freq and other norms than the 2-norm need backend = \"composite\"")
        if self.max_norm is not None:
            renorm_rows_(self.weight, idx, self.max_norm)
        return _ops.lookup_rows(w, idx, self.scale, self.padding_idx, 2 if self.sparse else 0)         # (2: padding stays on its own row)


# ---- dense layer in 16 bits --------------------------------------------------------------------------------------------------

def linear_act(x, weight, bias=None, activation="none", beta=1.0, residual=None):
    """activation(x weight^T + bias) + residual, all of it behind the product in the same pass: x [..., K], weight [N, K], bias [N],
    residual [..., N], all bf16 or all fp16 (fp32 layers run on the decoders' own dense tier); products accumulate in fp32.
    activation: "none", "relu", "silu", "gelu" (erf), "softplus" (with `beta`, as nn.Softplus).  No broadcasting: residual has the result's
    shape.  Up to 2^22 rows, N and K up to 2^20.  Differentiable once w.r.t. the four tensors.  Its gradients pass two roundings to the type
    beside those of its results: the value z before the activation is kept in 16 bits, which moves the slope a'(z) by up to a third of half
    a step (of 1, not of a'), and the gradient w.r.t. z is rounded before the two products that read it.  In fp16 the loss is scaled by
    the program, as for any fp16 layer."""
    act = _ACTIVATIONS.get("none" if activation is None else activation)
    if act is None:
        raise ValueError(f"linear_act: activation is one of {', '.join(_ACTIVATIONS)}, not {activation!r}")
    return _ops.linear_act(x, weight, bias, residual, act, beta)


# ---- global gradient norm ----------------------------------------------------------------------------------------------------

def _kind(what, norm_type):
    if norm_type == 2:
        return 0
    if norm_type == math.inf:
        return 1
    raise ValueError(f"{what}: norm_type is 2 or inf, not {norm_type}")


def _limit(what, max_norm):
    if not max_norm >= 0:
        raise ValueError(f"{what}: max_norm {max_norm}")
    return float(max_norm)


def grad_norm(grads, norm_type=2.0):
    """The 2-norm (squares added in fp64) or, with norm_type = inf, the largest magnitude over all tensors of `grads` (dense; fp32, bf16,
    fp16, mixed): a 0-dim fp32 tensor on their device, part of no graph."""
    kind = _kind("grad_norm", norm_type)
    grads = list(grads)
    return _ops.clip(grads, None, kind, 0.0, b"grad_norm") if grads else torch.zeros(())


def clip_grads(grads, max_norm, norm_type=2.0, out=None):
    """Scales the dense tensors of `grads` by min(1, max_norm / (norm + 1e-6)), in place, or into the tensors `out` (of the same sizes and types,
    in row-major order: pieces of a flat buffer will do).  A tensor that shares memory with another of the call, or is named twice, is
    refused.  -> (norm, the scaled tensors).  As torch's clip: a norm that is no number makes every result NaN, an infinite one makes the
    finite entries 0.  Norm and results are part of no graph.  Views with gaps go through a copy; strides so odd that it cannot be told in
    100 000 steps whether two views meet count as meeting."""
    what = "clip_grads"
    kind, limit = _kind(what, norm_type), _limit(what, max_norm)
    grads = list(grads)
    written = grads if out is None else list(out)
    if len(written) != len(grads):
        raise ValueError(f"{what}: {len(grads)} gradients, {len(written)} tensors in out")
    if not grads:
        return torch.zeros(()), written
    return _ops.clip(grads, written, kind, limit, what.encode()), written


def _merge_rows_(g):
    """Folds the duplicates of an uncoalesced row gradient, in place: the sum at a row's first entry, zeros at the others (same gradient)."""
    _ops.merge_rows_(g._indices()[0], g._values(), g.shape[0])


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ (training.py:128-131) with one norm over dense and row-sparse gradients: clips the ``.grad`` of `parameters`
    (a tensor or an iterable, none of them twice) in place and returns the norm before it (0-dim fp32).  Sparse gradients have one sparse
    dimension; entries that name the same row count as their sum, in the gradient's type (as it stays in the gradient).  One that is not coalesced and has rows of more than 256 entries is
    replaced by its coalesced form (as ``LatentCodes`` does; waits for the device, not while a graph is captured).
    ``error_if_nonfinite`` waits for the device and raises before anything is scaled."""
    what = "clip_grad_norm_"
    kind, limit = _kind(what, norm_type), _limit(what, max_norm)
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = []
    for p in parameters:
        g = p.grad
        if g is None:
            continue
        if g.is_sparse:
            if g.sparse_dim() != 1:
                raise ValueError(f"{what}: sparse gradients of whole rows (one sparse dimension)")
            v = g._values()
            if not (v.is_cuda and v.dtype in _CODES):
                raise TypeError(f"{what}: sparse fp32, bf16 or fp16 gradients on a ROCm device")
            if _needs_fold(g):
                p.grad = _folded(g)
                v = p.grad._values()
            elif not g.is_coalesced():
                _merge_rows_(g)
            g = v
        grads.append(g)
    if not grads:
        return torch.zeros(())
    if error_if_nonfinite:
        norm = _ops.clip(grads, None, kind, 0.0, what.encode())
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"{what}: the norm of the gradients is {float(norm)}; none was scaled")
    return _ops.clip(grads, grads, kind, limit, what.encode())
