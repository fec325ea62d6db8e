"""Operators of a training step around the decoders: the table of latent codes and its gradient, the dense layer in 16-bit storage
with its epilogue, the global gradient norm and clipping (what scripts/training/train.py does with nn.Embedding, nn.Linear and
clip_grad_norm_ between ``compute_loss`` and the optimisers, src/NPHM/models/training.py:111-135).

    codes = LatentCodes(n_subjects, 1344, max_norm=1.0, sparse=True, device="cuda")      # an nn.Embedding: same state_dict
    loss = weighted_total(compute_loss(batch, decoder, codes, device), lambdas)
    loss.backward()
    clip_grad_norm_(decoder.parameters(), 0.1)
    clip_grad_norm_(codes.parameters(), 0.1)                                            # row gradients too

Every function runs on libnphm_amd.so (csrc/rows_kernels.hip, clip_kernels.hip, layer16_kernels.hip), on the current stream of its
tensors' device, raises ``ValueError`` / ``TypeError`` for what it does not take and ``NphmAmdError`` if the library is missing; there is
no PyTorch fallback, CPU tensors are refused.  Results are the same bits from run to run.  All of it can be captured into a
graph, except where a line says that it waits for the device."""
from __future__ import annotations

import ctypes
import math

import torch
import torch.nn as nn

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "softplus": 4}


class _on:
    """Launches go to the current stream of `device`, which need not be the current device."""

    def __init__(self, device):
        self.device = device
        self.other = device.index is not None and device.index != torch.cuda.current_device()

    def __enter__(self):
        if self.other:
            self.before = torch.cuda.current_device()
            torch.cuda.set_device(self.device)
        return torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *exc):
        if self.other:
            torch.cuda.set_device(self.before)


def _need(cond, msg, kind=ValueError):
    if not cond:
        raise kind(msg)


def _on_gpu(what, t):
    _need(isinstance(t, torch.Tensor) and t.is_cuda, f"{what}: a tensor on a ROCm device (these operators have no CPU form)", TypeError)


# ---- rows of a table ---------------------------------------------------------------------------------------------------------

def _check_index(what, idx, device):
    _need(isinstance(idx, torch.Tensor) and idx.dtype in (torch.int32, torch.int64), f"{what}: idx is an int32 or int64 tensor", TypeError)
    _need(idx.device == device, f"{what}: idx is on {idx.device}, the rows on {device}")


def _padding(what, padding_idx, rows):
    if padding_idx is None:
        return -1
    _need(-rows <= padding_idx < rows, f"{what}: padding_idx {padding_idx} is no row of {rows}")
    return padding_idx % rows


def _row_strided(t):
    """(t or a copy of it, elements between its rows): rows contiguous, at least a row apart"""
    if t.shape[0] <= 1 or t.shape[1] == 0 or not (t.stride(1) == 1 or t.shape[1] == 1) or t.stride(0) < t.shape[1]:
        t = t.contiguous()
        return t, max(t.shape[1], 1)
    return t, t.stride(0)


def _lookup(table, idx, scale):
    rows, ld = _row_strided(table.detach())
    i = idx.contiguous()
    out = torch.empty(*idx.shape, table.shape[1], dtype=table.dtype, device=table.device)
    with _on(table.device) as stream:
        _lib.check(_lib.load().nphm_rows_lookup(rows.data_ptr(), rows.shape[0], rows.shape[1], ld, _DTYPES[table.dtype], i.data_ptr(),
                                                8 * i.element_size(), i.numel(), scale, out.data_ptr(), stream), "nphm_rows_lookup")
    return out


def lookup_rows_grad(grad, idx, num_rows, scale=1.0, padding_idx=None):
    """Gradient of ``lookup_rows`` w.r.t. its table of `num_rows` rows: [num_rows, D] of grad's type, ``scale`` times the sum of the rows
    of `grad` [*idx.shape, D] that name a row; zeros in rows that none names and in row `padding_idx`.  Sums are in fp32, in the
    order of the indices.  For programs that keep their own backward pass; autograd calls it by itself."""
    what = "lookup_rows_grad"
    _on_gpu(what, grad)
    _check_index(what, idx, grad.device)
    _need(grad.dtype in _DTYPES, f"{what}: fp32, bf16 or fp16 rows, not {grad.dtype}", TypeError)
    _need(grad.dim() >= 1 and grad.shape[:-1] == idx.shape, f"{what}: grad {tuple(grad.shape)} does not fit idx {tuple(idx.shape)}")
    _need(num_rows >= 1 and grad.shape[-1] >= 1, f"{what}: an empty table")
    _need(math.isfinite(scale), f"{what}: scale {scale}")
    pad = _padding(what, padding_idx, num_rows)
    D = grad.shape[-1]
    g, ld = _row_strided(grad.detach().reshape(-1, D))
    i = idx.contiguous()
    out = torch.empty(num_rows, D, dtype=grad.dtype, device=grad.device)
    lib = _lib.load()
    need = lib.nphm_rows_grad_workspace_bytes(num_rows, D, i.numel(), _DTYPES[grad.dtype])
    with _on(grad.device) as stream:
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device=grad.device)
        _lib.check(lib.nphm_rows_grad(g.data_ptr(), i.numel(), D, ld, _DTYPES[grad.dtype], i.data_ptr(), 8 * i.element_size(), num_rows, pad,
                                      scale, out.data_ptr(), ws.data_ptr(), need, stream), "nphm_rows_grad")
    return out


class _LookupFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, idx, scale, padding_idx, sparse):
        ctx.save_for_backward(idx)
        ctx.meta = (table.shape, scale, padding_idx, sparse)
        return _lookup(table, idx, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        (idx,) = ctx.saved_tensors
        (rows, D), scale, padding_idx, sparse = ctx.meta
        if not sparse:
            return lookup_rows_grad(g, idx, rows, scale, padding_idx), None, None, None, None
        # one entry an index, as nn.Embedding(sparse=True) leaves it; an entry that must not count names a row that exists and adds zeros
        i = idx.reshape(-1).long()
        keep = (i >= 0) & (i < rows)
        if padding_idx is not None:
            keep &= i != padding_idx % rows
        values = torch.where(keep[:, None], g.reshape(-1, D) * scale, torch.zeros((), dtype=g.dtype, device=g.device))
        return torch.sparse_coo_tensor(torch.where(keep, i, torch.zeros_like(i))[None], values, (rows, D), check_invariants=False), None, None, None, None


def lookup_rows(table, idx, scale=1.0, padding_idx=None, sparse=False):
    """scale * table[idx] for a table [V, D] (fp32, bf16 or fp16) and int32 / int64 indices of any shape: [*idx.shape, D] in the table's type,
    the product in fp32.  Differentiable (once) w.r.t. the table: a dense gradient (``lookup_rows_grad``) or, with ``sparse``, a
    sparse one with an entry for every index.  Row `padding_idx` is read like any other and gets no gradient.  An index outside
    the table gives a row of NaN and adds nothing to the gradient (nothing on the host looks at the indices)."""
    what = "lookup_rows"
    _on_gpu(what, table)
    _check_index(what, idx, table.device)
    _need(table.dtype in _DTYPES, f"{what}: a table of fp32, bf16 or fp16, not {table.dtype}", TypeError)
    _need(table.dim() == 2 and table.shape[0] >= 1 and table.shape[1] >= 1, f"{what}: a table [rows, width], not {tuple(table.shape)}")
    _need(math.isfinite(scale), f"{what}: scale {scale}")
    _padding(what, padding_idx, table.shape[0])
    if torch.is_grad_enabled() and table.requires_grad:
        return _LookupFn.apply(table, idx, float(scale), padding_idx, bool(sparse))
    return _lookup(table, idx, scale)


def renorm_rows_(table, idx, max_norm):
    """Rows of `table` that `idx` names and whose 2-norm is above `max_norm` are scaled down to it, in place, each once
    (nn.Embedding's max_norm, training.py:36-40)."""
    what = "renorm_rows_"
    _on_gpu(what, table)
    _check_index(what, idx, table.device)
    _need(table.dtype in _DTYPES, f"{what}: a table of fp32, bf16 or fp16, not {table.dtype}", TypeError)
    _need(table.dim() == 2 and table.shape[0] >= 1 and table.shape[1] >= 1 and (table.stride(1) == 1 or table.shape[1] == 1)
          and (table.shape[0] == 1 or table.stride(0) >= table.shape[1]), f"{what}: a table [rows, width] with contiguous rows")
    _need(max_norm >= 0, f"{what}: max_norm {max_norm}")
    i = idx.contiguous()
    with _on(table.device) as stream:
        flags = torch.empty(table.shape[0], dtype=torch.uint8, device=table.device)
        _lib.check(_lib.load().nphm_rows_renorm(table.data_ptr(), table.shape[0], table.shape[1], max(table.stride(0), table.shape[1]),
                                                _DTYPES[table.dtype], i.data_ptr(), 8 * i.element_size(), i.numel(), float(max_norm),
                                                flags.data_ptr(), stream), "nphm_rows_renorm")
    torch.autograd.graph.increment_version(table.detach())
    return table


class LatentCodes(nn.Embedding):
    """The table of latent codes of the trainers (nn.Embedding(n, lat_dim, max_norm=1.0, sparse=True), training.py:36-40) on
    ``lookup_rows`` / ``renorm_rows_``; parameters, initialisation and state_dict are nn.Embedding's.  ``scale`` multiplies the looked-up
    rows.  ``backend = "composite"`` computes the same with torch's embedding (CPU tensors need it, as in the decoders)."""

    def __init__(self, num_embeddings, embedding_dim, padding_idx=None, max_norm=None, scale=1.0, sparse=False, device=None, dtype=None):
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx, max_norm=max_norm, sparse=sparse, device=device, dtype=dtype)
        _need(math.isfinite(scale), f"LatentCodes: scale {scale}")
        self.scale = float(scale)
        self.backend = "hip"            # "hip" | "composite"

    def forward(self, idx):
        if self.backend == "composite":
            rows = super().forward(idx)
            return rows if self.scale == 1.0 else rows * self.scale
        if self.max_norm is not None:
            renorm_rows_(self.weight, idx, self.max_norm)
        return lookup_rows(self.weight, idx, self.scale, self.padding_idx, self.sparse)


# ---- dense layer in 16 bits --------------------------------------------------------------------------------------------------

def _workspace(nbytes, device):
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device)


class _LinearActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, beta, keep):
        lib = _lib.load()
        x2, w = x.detach().reshape(-1, x.shape[-1]).contiguous(), weight.detach().contiguous()
        M, K = x2.shape
        N = w.shape[0]
        y = torch.empty(*x.shape[:-1], N, dtype=x.dtype, device=x.device)
        z = torch.empty(M, N, dtype=x.dtype, device=x.device) if keep and act else None
        if M:
            b = None if bias is None else bias.detach().contiguous()
            r = None if residual is None else residual.detach().contiguous()
            with _on(x.device) as stream:
                need = lib.nphm_layer16_forward_workspace_bytes(M, N, K)
                ws = _workspace(need, x.device)
                _lib.check(lib.nphm_layer16_forward(x2.data_ptr(), w.data_ptr(), None if b is None else b.data_ptr(),
                                                    None if r is None else r.data_ptr(), y.data_ptr(), None if z is None else z.data_ptr(),
                                                    M, N, K, _DTYPES[x.dtype], act, beta, ws.data_ptr(), need, stream), "nphm_layer16_forward")
        if keep:
            ctx.save_for_backward(x, weight, z)
            ctx.meta = (act, beta, bias is not None)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        lib = _lib.load()
        x, weight, z = ctx.saved_tensors
        act, beta, _ = ctx.meta
        x2, w = x.detach().reshape(-1, x.shape[-1]).contiguous(), weight.detach().contiguous()
        M, K = x2.shape
        N = w.shape[0]
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        new = torch.empty if M else torch.zeros
        dx = new(x.shape, dtype=x.dtype, device=x.device) if need_x else None
        dw = new(N, K, dtype=x.dtype, device=x.device) if need_w else None
        db = new(N, dtype=x.dtype, device=x.device) if need_b else None
        if M and (need_x or need_w or need_b):
            g2 = g.reshape(M, N).contiguous()
            with _on(x.device) as stream:
                need = lib.nphm_layer16_backward_workspace_bytes(M, N, K, act)
                ws = _workspace(need, x.device)
                p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
                _lib.check(lib.nphm_layer16_backward(g2.data_ptr(), x2.data_ptr(), w.data_ptr(), p(z), p(dx), p(dw), p(db), M, N, K,
                                                     _DTYPES[x.dtype], act, beta, ws.data_ptr(), need, stream), "nphm_layer16_backward")
        return dx, dw, db, g if need_r else None, None, None, None


def linear_act(x, weight, bias=None, activation="none", beta=1.0, residual=None):
    """activation(x weight^T + bias) + residual in one launch: x [..., K], weight [N, K], bias [N], residual [..., N], all bf16 or all fp16 (fp32
    layers run on the decoders' own dense tier); products accumulate in fp32.  activation: "none", "relu", "silu", "gelu"
    (erf), "softplus" (with `beta`, as nn.Softplus).  Differentiable once w.r.t. the four tensors: the value before the activation is
    kept in 16 bits for it.  No broadcasting: residual has the result's shape."""
    what = "linear_act"
    _on_gpu(what, x)
    _need(x.dtype in (torch.bfloat16, torch.float16), f"{what}: bf16 or fp16 tensors, not {x.dtype}", TypeError)
    _need(x.dim() >= 1 and weight.dim() == 2 and x.shape[-1] == weight.shape[1] and weight.shape[0] >= 1 and weight.shape[1] >= 1,
          f"{what}: x {tuple(x.shape)} does not fit weight {tuple(weight.shape)}")
    N = weight.shape[0]
    _need(bias is None or tuple(bias.shape) == (N,), f"{what}: bias has the shape ({N},)")
    _need(residual is None or tuple(residual.shape) == (*x.shape[:-1], N), f"{what}: residual has the shape of the result")
    for t in (weight, bias, residual):
        _need(t is None or (t.device == x.device and t.dtype == x.dtype), f"{what}: all tensors on one device, of one type", TypeError)
    act = _ACTIVATIONS.get("none" if activation is None else activation)
    _need(act is not None, f"{what}: activation is one of {', '.join(_ACTIVATIONS)}, not {activation!r}")
    _need(act != 4 or (math.isfinite(beta) and beta > 0), f"{what}: Softplus takes a positive beta, not {beta}")
    keep = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual))
    return _LinearActFn.apply(x, weight, bias, residual, act, float(beta), keep)


# ---- global gradient norm ----------------------------------------------------------------------------------------------------

def _kind(what, norm_type):
    norm_type = float(norm_type)
    _need(norm_type in (2.0, math.inf), f"{what}: norm_type is 2 or inf, not {norm_type}")
    return 0 if norm_type == 2.0 else 1


def _flat_order(t):
    """the order of t's dimensions in memory if t fills its span of memory without gaps or repeats, else None"""
    order = sorted((d for d in range(t.dim()) if t.shape[d] != 1), key=t.stride, reverse=True)
    want = 1
    for d in reversed(order):
        if t.stride(d) != want:
            return None
        want *= t.shape[d]
    return order


def _clip(what, grads, out, kind, limit):
    """-> norm; out None: the norm alone"""
    dev = grads[0].device
    ins, outs, back = [], [], []
    for k, g in enumerate(grads):
        _on_gpu(what, g)
        _need(g.dtype in _DTYPES, f"{what}: fp32, bf16 or fp16 gradients, not {g.dtype}", TypeError)
        _need(g.device == dev, f"{what}: gradients on {dev} and {g.device}: one call takes one device's")
        o = None if out is None else out[k]
        if o is not None and o is not g:
            _need(isinstance(o, torch.Tensor) and o.shape == g.shape and o.dtype == g.dtype and o.device == g.device,
                  f"{what}: out has a tensor of the shape, type and device of each gradient")
        if not g.is_contiguous() or (o is not None and o is not g and not o.is_contiguous()):
            order = None if g.numel() == 0 else _flat_order(g)
            if order is None or not (o is None or o is g or o.stride() == g.stride()):
                g = g.contiguous()
                if o is not None:
                    o_flat = torch.empty_like(g)
                    back.append((o, o_flat))
                    o = o_flat
        ins.append(g)
        outs.append(o)
    n = len(ins)
    lib = _lib.load()
    counts = (ctypes.c_int64 * n)(*[g.numel() for g in ins])
    dtypes = (ctypes.c_int * n)(*[_DTYPES[g.dtype] for g in ins])
    p_in = (ctypes.c_void_p * n)(*[g.data_ptr() for g in ins])
    p_out = None if out is None else (ctypes.c_void_p * n)(*[o.data_ptr() for o in outs])
    with _on(dev) as stream:
        need = lib.nphm_clip_workspace_bytes(counts, n)
        ws = _workspace(need, dev)
        norm = torch.empty((), dtype=torch.float32, device=dev)
        _lib.check(lib.nphm_clip_grads(p_in, p_out, counts, dtypes, n, kind, limit, norm.data_ptr(), ws.data_ptr(), need, stream),
                   "nphm_clip_grads")
    for o, o_flat in back:
        o.copy_(o_flat)
    if out is not None:
        torch.autograd.graph.increment_version([o for o in out])
    return norm


def _detached(tensors):
    return [t.detach() if isinstance(t, torch.Tensor) and t.requires_grad else t for t in tensors]


def grad_norm(grads, norm_type=2.0):
    """The 2-norm (squares added in fp64) or, with norm_type = inf, the largest magnitude over all tensors of `grads` (dense; fp32, bf16,
    fp16, mixed): a 0-dim fp32 tensor on their device."""
    kind = _kind("grad_norm", norm_type)
    grads = _detached(grads)
    if not grads:
        return torch.zeros(())
    return _clip("grad_norm", grads, None, kind, 0.0)


def clip_grads(grads, max_norm, norm_type=2.0, out=None):
    """Scales the dense tensors of `grads` by min(1, max_norm / (norm + 1e-6)), in place, or into the tensors `out` (same shapes and types, of
    which none shares memory with another tensor of the call).  -> (norm, the scaled tensors).  As torch's clip: a norm that is
    no number makes every result NaN, an infinite one makes the finite entries 0."""
    what = "clip_grads"
    kind = _kind(what, norm_type)
    _need(max_norm >= 0, f"{what}: max_norm {max_norm}")
    grads = list(grads)
    written = grads if out is None else list(out)
    _need(len(written) == len(grads), f"{what}: {len(grads)} gradients, {len(written)} tensors in out")
    if not grads:
        return torch.zeros(()), written
    src = _detached(grads)
    norm = _clip(what, src, src if out is None else _detached(written), kind, float(max_norm))
    return norm, written


def _merge_rows_(g):
    """Folds the duplicates of an uncoalesced row gradient, in place: the sum at a row's first entry, zeros at the others (same gradient)."""
    i, v = g._indices()[0].contiguous(), g._values()
    flat = v.reshape(v.shape[0], -1).contiguous()
    if flat.numel() == 0:
        return
    out = torch.empty_like(flat)
    lib = _lib.load()
    need = lib.nphm_rows_grad_workspace_bytes(g.shape[0], flat.shape[1], flat.shape[0], _DTYPES[v.dtype])
    with _on(v.device) as stream:
        ws = _workspace(need, v.device)
        _lib.check(lib.nphm_rows_merge(flat.data_ptr(), flat.shape[0], flat.shape[1], _DTYPES[v.dtype], i.data_ptr(), 64, g.shape[0],
                                       out.data_ptr(), ws.data_ptr(), need, stream), "nphm_rows_merge")
    v.copy_(out.view_as(v))


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ (training.py:128-131) with one norm over dense and row-sparse gradients: clips the ``.grad`` of `parameters`
    (a tensor or an iterable) in place and returns the norm before it (0-dim fp32).  Sparse gradients have one sparse dimension;
    entries that name the same row count as their sum.  ``error_if_nonfinite`` waits for the device and raises before
    anything is scaled."""
    what = "clip_grad_norm_"
    kind = _kind(what, norm_type)
    _need(max_norm >= 0, f"{what}: max_norm {max_norm}")
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = []
    for g in [p.grad for p in parameters if p.grad is not None]:
        if g.is_sparse:
            _need(g.sparse_dim() == 1, f"{what}: sparse gradients of whole rows (one sparse dimension)")
            _need(g._values().is_cuda and g._values().dtype in _DTYPES, f"{what}: sparse fp32, bf16 or fp16 gradients on a ROCm device", TypeError)
            if not g.is_coalesced():
                _merge_rows_(g.detach())
            g = g.detach()._values()
        grads.append(g)
    if not grads:
        return torch.zeros(())
    grads = _detached(grads)
    if error_if_nonfinite:
        norm = _clip(what, grads, None, kind, 0.0)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"{what}: the norm of the gradients is {float(norm)}; none was scaled")
    return _clip(what, grads, grads, kind, float(max_norm))
