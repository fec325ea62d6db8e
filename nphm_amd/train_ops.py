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

import math
from array import array
from operator import attrgetter

import torch
import torch.nn as nn

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "softplus": 4}


_raw_stream = torch._C._cuda_getCurrentRawStream        # (torch.cuda.current_stream builds an object around it: 2 us a call)


class _on:
    """Makes `device` the current one for the launches inside and yields the handle of its current stream (the tensors' device need not
    be the current one)."""

    def __init__(self, device):
        self.index = device.index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return _raw_stream(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


def _workspace(nbytes, device):
    """-> (tensor or None, its address or None)"""
    if not nbytes:
        return None, None
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr()


def _written(tensors):
    """tells autograd that the tensors were written (inference tensors keep no version)"""
    try:
        torch.autograd.graph.increment_version(tensors)
    except RuntimeError:
        torch.autograd.graph.increment_version([t for t in tensors if not t.is_inference()])


def _on_gpu(what, t):
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise TypeError(f"{what}: a tensor on a ROCm device (these operators have no CPU form)")


# ---- rows of a table ---------------------------------------------------------------------------------------------------------

def _check_rows(what, rows, idx, scale):
    """rows and indices that fit each other, on a ROCm device"""
    _on_gpu(what, rows)
    if rows.dtype not in _DTYPES:
        raise TypeError(f"{what}: rows of fp32, bf16 or fp16, not {rows.dtype}")
    if not isinstance(idx, torch.Tensor) or idx.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{what}: idx is an int32 or int64 tensor")
    if idx.device != rows.device:
        raise ValueError(f"{what}: idx is on {idx.device}, the rows on {rows.device}")
    if not math.isfinite(scale):
        raise ValueError(f"{what}: scale {scale}")


def _check_table(what, table):
    if table.dim() != 2 or table.numel() == 0:
        raise ValueError(f"{what}: a table [rows, width], not {tuple(table.shape)}")


def _padding(what, padding_idx, rows):
    if padding_idx is None:
        return -1
    if not -rows <= padding_idx < rows:
        raise ValueError(f"{what}: padding_idx {padding_idx} is no row of {rows}")
    return padding_idx % rows


def _row_strided(t):
    """(t or a copy of it, elements between its rows): rows contiguous, at least a row apart"""
    if t.is_contiguous():
        return t, t.shape[1]
    if t.stride(1) != 1 or t.stride(0) < t.shape[1]:
        t = t.contiguous()
        return t, t.shape[1]
    return t, t.stride(0)


def _lookup(table, idx, scale):
    rows, ld = _row_strided(table)
    V, D = table.shape
    i = idx if idx.is_contiguous() else idx.contiguous()
    out = torch.empty((*idx.shape, D), dtype=table.dtype, device=table.device)
    with _on(table.device) as stream:
        rc = _lib.load().nphm_rows_lookup(rows.data_ptr(), V, D, ld, _DTYPES[table.dtype], i.data_ptr(), 64 if i.dtype == torch.int64 else 32,
                                          i.numel(), scale, out.data_ptr(), stream)
    if rc:
        _lib.check(rc, "nphm_rows_lookup")
    return out


@torch.no_grad()
def lookup_rows_grad(grad, idx, num_rows, scale=1.0, padding_idx=None):
    """Gradient of ``lookup_rows`` w.r.t. its table of `num_rows` rows: [num_rows, D] of grad's type, ``scale`` times the sum of the rows
    of `grad` [*idx.shape, D] that name a row; zeros in rows that none names and in row `padding_idx`.  Sums are in fp32, in the
    order of the indices.  For programs that keep their own backward pass; autograd calls it by itself."""
    what = "lookup_rows_grad"
    _check_rows(what, grad, idx, scale)
    if grad.dim() < 1 or grad.shape[:-1] != idx.shape:
        raise ValueError(f"{what}: grad {tuple(grad.shape)} does not fit idx {tuple(idx.shape)}")
    D, scale = grad.shape[-1], float(scale)
    if num_rows < 1 or D < 1:
        raise ValueError(f"{what}: an empty table")
    pad = _padding(what, padding_idx, num_rows)
    g, ld = _row_strided(grad if grad.dim() == 2 else grad.reshape(-1, D))
    i = idx if idx.is_contiguous() else idx.contiguous()
    count, code = i.numel(), _DTYPES[grad.dtype]
    out = torch.empty((num_rows, D), dtype=grad.dtype, device=grad.device)
    lib = _lib.load()
    need = lib.nphm_rows_grad_workspace_bytes(num_rows, D, count, code)
    with _on(grad.device) as stream:
        ws, at = _workspace(need, grad.device)
        rc = lib.nphm_rows_grad(g.data_ptr(), count, D, ld, code, i.data_ptr(), 64 if i.dtype == torch.int64 else 32, num_rows, pad, scale,
                                out.data_ptr(), at, need, stream)
    if rc:
        _lib.check(rc, "nphm_rows_grad")
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
    _check_rows(what, table, idx, scale)
    _check_table(what, table)
    if padding_idx is not None:
        _padding(what, padding_idx, table.shape[0])
    if table.requires_grad and torch.is_grad_enabled():
        return _LookupFn.apply(table, idx, float(scale), padding_idx, bool(sparse))
    return _lookup(table, idx, float(scale))


def renorm_rows_(table, idx, max_norm):
    """Rows of `table` that `idx` names and whose 2-norm is above `max_norm` are scaled down to it, in place, each once
    (nn.Embedding's max_norm, training.py:36-40)."""
    what = "renorm_rows_"
    _check_rows(what, table, idx, 1.0)
    _check_table(what, table)
    V, D = table.shape
    if (D > 1 and table.stride(1) != 1) or (V > 1 and table.stride(0) < D):
        raise ValueError(f"{what}: a table with contiguous rows")
    if not max_norm >= 0:
        raise ValueError(f"{what}: max_norm {max_norm}")
    i = idx if idx.is_contiguous() else idx.contiguous()
    with _on(table.device) as stream:
        flags = torch.empty(V, dtype=torch.uint8, device=table.device)
        rc = _lib.load().nphm_rows_renorm(table.data_ptr(), V, D, max(table.stride(0), D), _DTYPES[table.dtype], i.data_ptr(),
                                          64 if i.dtype == torch.int64 else 32, i.numel(), float(max_norm), flags.data_ptr(), stream)
    if rc:
        _lib.check(rc, "nphm_rows_renorm")
    _written([table.detach()])
    return table


class LatentCodes(nn.Embedding):
    """The table of latent codes of the trainers (nn.Embedding(n, lat_dim, max_norm=1.0, sparse=True), training.py:36-40) on
    ``lookup_rows`` / ``renorm_rows_``; parameters, initialisation and state_dict are nn.Embedding's.  ``scale`` multiplies the looked-up
    rows.  ``backend = "composite"`` computes the same with torch's embedding (CPU tensors need it, as in the decoders)."""

    def __init__(self, num_embeddings, embedding_dim, padding_idx=None, max_norm=None, scale=1.0, sparse=False, device=None, dtype=None):
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx, max_norm=max_norm, sparse=sparse, device=device, dtype=dtype)
        if not math.isfinite(scale):
            raise ValueError(f"LatentCodes: scale {scale}")
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

def _rows_of(t):
    """t as contiguous rows [M, K]"""
    t = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    return t if t.is_contiguous() else t.contiguous()


def _layer_forward(x, weight, bias, residual, act, beta, keep):
    """-> (y, z or None)"""
    x2, w = _rows_of(x), weight if weight.is_contiguous() else weight.contiguous()
    M, K = x2.shape
    N = w.shape[0]
    y = torch.empty((*x.shape[:-1], N), dtype=x.dtype, device=x.device)
    z = torch.empty((M, N), dtype=x.dtype, device=x.device) if keep and act else None
    if M:
        b = None if bias is None else bias.contiguous()
        r = None if residual is None else residual.contiguous()
        lib = _lib.load()
        with _on(x.device) as stream:
            need = lib.nphm_layer16_forward_workspace_bytes(x2.data_ptr(), w.data_ptr(), M, N, K)
            ws, at = _workspace(need, x.device)
            rc = lib.nphm_layer16_forward(x2.data_ptr(), w.data_ptr(), None if b is None else b.data_ptr(), None if r is None else r.data_ptr(),
                                          y.data_ptr(), None if z is None else z.data_ptr(), M, N, K, _DTYPES[x.dtype], act, beta, at, need, stream)
        if rc:
            _lib.check(rc, "nphm_layer16_forward")
    return y, z


class _LinearActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, beta):
        y, z = _layer_forward(x, weight, bias, residual, act, beta, True)
        ctx.save_for_backward(x, weight, z)
        ctx.meta = (act, beta)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, weight, z = ctx.saved_tensors
        act, beta = ctx.meta
        x2, w = _rows_of(x), weight if weight.is_contiguous() else weight.contiguous()
        M, K = x2.shape
        N = w.shape[0]
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        new = torch.empty if M else torch.zeros
        dx = new(x.shape, dtype=x.dtype, device=x.device) if need_x else None
        dw = new((N, K), dtype=x.dtype, device=x.device) if need_w else None
        db = new((N,), dtype=x.dtype, device=x.device) if need_b else None
        if M and (need_x or need_w or need_b):
            g2 = _rows_of(g)
            lib = _lib.load()
            with _on(x.device) as stream:
                need = lib.nphm_layer16_backward_workspace_bytes(g2.data_ptr(), x2.data_ptr(), w.data_ptr(), M, N, K, act)
                ws, at = _workspace(need, x.device)
                rc = lib.nphm_layer16_backward(g2.data_ptr(), x2.data_ptr(), w.data_ptr(), None if z is None else z.data_ptr(),
                                               None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(),
                                               None if db is None else db.data_ptr(), M, N, K, _DTYPES[x.dtype], act, beta, at, need, stream)
            if rc:
                _lib.check(rc, "nphm_layer16_backward")
        return dx, dw, db, g if need_r else None, None, None


def linear_act(x, weight, bias=None, activation="none", beta=1.0, residual=None):
    """activation(x weight^T + bias) + residual in one launch: x [..., K], weight [N, K], bias [N], residual [..., N], all bf16 or all fp16 (fp32
    layers run on the decoders' own dense tier); products accumulate in fp32.  activation: "none", "relu", "silu", "gelu"
    (erf), "softplus" (with `beta`, as nn.Softplus).  Differentiable once w.r.t. the four tensors: the value before the activation is
    kept in 16 bits for it.  No broadcasting: residual has the result's shape."""
    what = "linear_act"
    _on_gpu(what, x)
    t, dev = x.dtype, x.device
    if t not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{what}: bf16 or fp16 tensors, not {t}")
    _on_gpu(what, weight)
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or weight.numel() == 0:
        raise ValueError(f"{what}: x {tuple(x.shape)} does not fit weight {tuple(weight.shape)}")
    N = weight.shape[0]
    if bias is not None and bias.shape != (N,):
        raise ValueError(f"{what}: bias has the shape ({N},)")
    if residual is not None and residual.shape != (*x.shape[:-1], N):
        raise ValueError(f"{what}: residual has the shape of the result")
    grad = x.requires_grad
    for o in (weight, bias, residual):
        if o is not None:
            if o.dtype != t or o.device != dev:
                raise TypeError(f"{what}: all tensors on one device, of one type")
            grad = grad or o.requires_grad
    act = _ACTIVATIONS.get("none" if activation is None else activation)
    if act is None:
        raise ValueError(f"{what}: activation is one of {', '.join(_ACTIVATIONS)}, not {activation!r}")
    if act == 4 and not (math.isfinite(beta) and beta > 0):
        raise ValueError(f"{what}: Softplus takes a positive beta, not {beta}")
    if grad and torch.is_grad_enabled():
        return _LinearActFn.apply(x, weight, bias, residual, act, float(beta))
    return _layer_forward(x, weight, bias, residual, act, float(beta), False)[0]


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


def _gapless(t):
    """whether t fills its span of memory without gaps or repeats, whatever the order of its dimensions"""
    want = 1
    for n, stride in sorted(((t.shape[d], t.stride(d)) for d in range(t.dim()) if t.shape[d] != 1), key=lambda v: v[1]):
        if stride != want:
            return False
        want *= n
    return True


_Tensor = torch.Tensor
_dtype_of = attrgetter("dtype")


@torch.no_grad()
def _clip(what, grads, out, kind, limit):
    """-> norm; out None: the norm alone.  (A list may hold hundreds of tensors, and a look at each of them costs 0.1 us a question: they are
    asked as few as will do, by maps, and one by one only where something is to be said or done about one.)"""
    apart = out is not None and out is not grads
    for tensors in (grads, out) if apart else (grads,):
        if not set(map(type, tensors)) <= {_Tensor, nn.Parameter}:
            for t in tensors:
                _on_gpu(what, t)
    n = len(grads)
    devices, types = set(map(_Tensor.get_device, grads)), set(map(_dtype_of, grads))
    if len(devices) != 1 or -1 in devices:
        for g in grads:
            _on_gpu(what, g)
        raise ValueError(f"{what}: gradients on {len(devices)} devices: one call takes one device's")
    if not types <= _DTYPES.keys():
        raise TypeError(f"{what}: fp32, bf16 or fp16 gradients, not {', '.join(map(str, types - _DTYPES.keys()))}")
    one = len(types) == 1
    codes = array("i", [_DTYPES[types.pop()]]) * n if one else array("i", [_DTYPES[t] for t in map(_dtype_of, grads)])
    counts = array("q", map(_Tensor.numel, grads))
    plain = all(map(_Tensor.is_contiguous, grads))
    if apart:
        if (array("q", map(_Tensor.numel, out)) != counts or set(map(_Tensor.get_device, out)) != devices
                or (set(map(_dtype_of, out)) != {grads[0].dtype} if one else list(map(_dtype_of, out)) != list(map(_dtype_of, grads)))):
            raise ValueError(f"{what}: out has a tensor of the size, type and device of each gradient")
        plain = plain and all(map(_Tensor.is_contiguous, out))
    ins, outs, back = grads, out, []
    if not plain:
        ins, outs = list(grads), None if out is None else list(out)
        for k, g in enumerate(grads):
            o = g if out is None else out[k]
            if (g.is_contiguous() and o.is_contiguous()) or (g.shape == o.shape and g.stride() == o.stride() and _gapless(g)):
                continue                                             # (any order of dimensions, the same on both sides)
            ins[k] = g.contiguous()
            if out is not None:
                outs[k] = torch.empty_like(ins[k])
                back.append((o, outs[k]))
    p_in = array("Q", map(_Tensor.data_ptr, ins))
    p_out = None if out is None else p_in if outs is ins else array("Q", map(_Tensor.data_ptr, outs))
    dev = grads[0].device
    lib = _lib.load()
    at = lambda a: a.buffer_info()[0]  # noqa: E731
    with _on(dev) as stream:
        need = lib.nphm_clip_workspace_bytes(at(counts), n)
        ws, ws_at = _workspace(need, dev)
        norm = torch.empty((), dtype=torch.float32, device=dev)
        rc = lib.nphm_clip_grads(at(p_in), None if out is None else at(p_out), at(counts), at(codes), n, kind, limit, norm.data_ptr(), ws_at,
                                 need, stream)
    if rc:
        _lib.check(rc, "nphm_clip_grads")
    for o, flat in back:
        o.copy_(flat.view(o.shape))
    if out is not None:
        _written(out)
    return norm


def grad_norm(grads, norm_type=2.0):
    """The 2-norm (squares added in fp64) or, with norm_type = inf, the largest magnitude over all tensors of `grads` (dense; fp32, bf16,
    fp16, mixed): a 0-dim fp32 tensor on their device."""
    kind = _kind("grad_norm", norm_type)
    grads = list(grads)
    return _clip("grad_norm", grads, None, kind, 0.0) if grads else torch.zeros(())


def clip_grads(grads, max_norm, norm_type=2.0, out=None):
    """Scales the dense tensors of `grads` by min(1, max_norm / (norm + 1e-6)), in place, or into the tensors `out` (of the same sizes and types,
    in row-major order: pieces of a flat buffer will do; none shares memory with another tensor of the call).  -> (norm, the scaled tensors).  As torch's clip: a norm that is
    no number makes every result NaN, an infinite one makes the finite entries 0."""
    what = "clip_grads"
    kind, limit = _kind(what, norm_type), _limit(what, max_norm)
    grads = list(grads)
    written = grads if out is None else list(out)
    if len(written) != len(grads):
        raise ValueError(f"{what}: {len(grads)} gradients, {len(written)} tensors in out")
    if not grads:
        return torch.zeros(()), written
    return _clip(what, grads, written, kind, limit), written


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
        ws, at = _workspace(need, v.device)
        _lib.check(lib.nphm_rows_merge(flat.data_ptr(), flat.shape[0], flat.shape[1], _DTYPES[v.dtype], i.data_ptr(), 64, g.shape[0],
                                       out.data_ptr(), at, need, stream), "nphm_rows_merge")
    v.copy_(out.view_as(v))


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ (training.py:128-131) with one norm over dense and row-sparse gradients: clips the ``.grad`` of `parameters`
    (a tensor or an iterable) in place and returns the norm before it (0-dim fp32).  Sparse gradients have one sparse dimension;
    entries that name the same row count as their sum.  ``error_if_nonfinite`` waits for the device and raises before
    anything is scaled."""
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
            if not (v.is_cuda and v.dtype in _DTYPES):
                raise TypeError(f"{what}: sparse fp32, bf16 or fp16 gradients on a ROCm device")
            if not g.is_coalesced():
                _merge_rows_(g)
            g = v
        grads.append(g)
    if not grads:
        return torch.zeros(())
    if error_if_nonfinite:
        norm = _clip(what, grads, None, kind, 0.0)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"{what}: the norm of the gradients is {float(norm)}; none was scaled")
    return _clip(what, grads, grads, kind, limit)
