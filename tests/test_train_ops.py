"""The training operators (nphm_amd.train_ops) against plain forms in 64 bits: rows of a table and their gradient, the 16-bit dense
layer and its gradients, the gradient norm and clipping, and a step that uses all of them.

Tolerances count roundings.  A rounding to a type moves a value by at most eps / 2 of it, ``torch.finfo(t).eps / 2``; a sum of n fp32 terms
by at most (n - 1) 2^-24 of the sum of their magnitudes (the matrix instructions' internal adds are taken as twice that)."""
import math

import numpy as np
import pytest
import torch

import _util as U
from nphm_amd import train_ops as T
from nphm_amd._lib import NphmAmdError
from nphm_amd.deepsdf import DeepSDF, _DenseLayerFn

gpu = pytest.mark.gpu
FLOATS = [torch.float32, torch.bfloat16, torch.float16]
HALVES = [torch.bfloat16, torch.float16]
F32 = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps       # the step below the smallest normal number


def within(got, want, bound):
    """|got - want| <= bound everywhere, all in fp64; says by how much the worst one misses or fits"""
    d = (got.double() - want).abs()
    assert bool(torch.isfinite(d).all()), "a value that is not finite"
    worst = float((d / bound.clamp(min=1e-300)).max()) if d.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} of the bound"
    return worst


# ---- refusals (no GPU is touched) -----------------------------------------------------------------------------------------------

def test_cpu_tensors_are_refused():
    t, i = torch.zeros(4, 8), torch.zeros(3, dtype=torch.long)
    for call in (lambda: T.lookup_rows(t, i), lambda: T.lookup_rows_grad(torch.zeros(3, 8), i, 4), lambda: T.renorm_rows_(t, i, 1.0),
                 lambda: T.linear_act(t.bfloat16(), t.bfloat16()), lambda: T.grad_norm([t]), lambda: T.clip_grads([t], 1.0)):
        with pytest.raises(TypeError):
            call()
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(TypeError):
        T.clip_grad_norm_([p], 1.0)


def test_module_on_cpu_needs_the_composite_backend():
    codes = T.LatentCodes(5, 8, max_norm=1.0, scale=2.0)
    with pytest.raises(TypeError):
        codes(torch.tensor([1, 2]))
    codes.backend = "composite"
    got = codes(torch.tensor([1, 2, 1]))
    assert torch.equal(got, 2.0 * codes.weight[torch.tensor([1, 2, 1])])
    assert float(codes.weight[1].detach().norm()) <= 1.0 + 1e-6
    other = torch.nn.Embedding(5, 8)
    other.load_state_dict(codes.state_dict())


def test_module_takes_what_an_embedding_takes():
    """from_pretrained and its arguments; what the kernels do not compute is refused, not left out"""
    rows = torch.randn(6, 5)
    codes = T.LatentCodes.from_pretrained(rows, freeze=False, padding_idx=-1, max_norm=0.5, norm_type=1.0, scale_grad_by_freq=True)
    assert isinstance(codes, T.LatentCodes) and codes.weight.requires_grad and codes.padding_idx == 5 and codes.scale == 1.0 and codes.weight.data_ptr() == rows.data_ptr()
    idx = torch.tensor([1, 5, 1, 2])
    with pytest.raises(ValueError, match="composite"):
        codes(idx)
    codes.backend = "composite"
    twin = torch.nn.Embedding.from_pretrained(rows.clone(), freeze=False, padding_idx=-1, max_norm=0.5, norm_type=1.0, scale_grad_by_freq=True)
    a, b = codes(idx), twin(idx)
    a.sum().backward()
    b.sum().backward()
    assert torch.equal(a, b) and torch.equal(codes.weight.grad, twin.weight.grad)
    frozen = T.LatentCodes.from_pretrained(rows)
    assert not frozen.weight.requires_grad and frozen.max_norm is None
    for codes in (T.LatentCodes(4, 3, scale_grad_by_freq=True), T.LatentCodes(4, 3, max_norm=1.0, norm_type=math.inf)):
        with pytest.raises(ValueError, match="composite"):
            codes(idx[:1])
    with pytest.raises(TypeError):                                  # the norm of rows that are not bounded matters to nobody: on to the device's check
        T.LatentCodes(4, 3, norm_type=1.0)(idx[:1])
    with pytest.raises(AssertionError):
        T.LatentCodes.from_pretrained(rows[0])


def test_bad_arguments_are_refused():
    for kind in (1.0, 3.0, 0.0):
        with pytest.raises(ValueError):
            T.grad_norm([], norm_type=kind)
    for limit in (-1.0, math.nan):
        with pytest.raises(ValueError):
            T.clip_grads([], limit)
        with pytest.raises(ValueError):
            T.clip_grad_norm_([], limit)
    with pytest.raises(ValueError):
        T.clip_grads([], 1.0, out=[torch.zeros(1)])
    assert float(T.grad_norm([])) == 0.0 and float(T.clip_grad_norm_([], 1.0)) == 0.0
    with pytest.raises(ValueError):
        T.LatentCodes(4, 8, scale=math.inf)


def test_c_entries_refuse_before_any_launch():
    """what the host can see is an error, not a launch: sizes, types, null pointers, memory that tensors share"""
    import ctypes
    from nphm_amd import _lib
    lib = _lib.load()
    assert lib.nphm_rows_lookup(None, 4, 8, 8, 0, None, 64, 1, 1.0, None, None) != 0
    assert lib.nphm_rows_lookup(16, 4, 8, 7, 0, 16, 64, 1, 1.0, 16, None) != 0 and b"stride" in lib.nphm_last_error()
    assert lib.nphm_rows_lookup(16, 4, 8, 8, 3, 16, 64, 1, 1.0, 16, None) != 0 and b"dtype" in lib.nphm_last_error()
    assert lib.nphm_rows_lookup(16, 4, 8, 8, 0, 16, 16, 1, 1.0, 16, None) != 0 and b"bits" in lib.nphm_last_error()
    assert lib.nphm_rows_grad(16, 1 << 27, 8, 8, 0, 16, 64, 4, -1, 1.0, 16, 16, 1 << 40, None) != 0 and b"sizes" in lib.nphm_last_error()
    assert lib.nphm_rows_renorm(16, 4, 8, 8, 0, 16, 64, 1, -1.0, 16, None) != 0 and b"max_norm" in lib.nphm_last_error()
    assert lib.nphm_layer16_forward(16, 16, None, None, 16, None, 4, 4, 4, 0, 0, 1.0, None, 0, None) != 0 and b"dtype" in lib.nphm_last_error()
    assert lib.nphm_layer16_forward(16, 16, None, None, 16, None, 0, 4, 4, 1, 0, 1.0, None, 0, None) != 0 and b"sizes" in lib.nphm_last_error()
    assert lib.nphm_layer16_forward(16, 16, None, None, 16, None, 4, 4, 4, 1, 9, 1.0, None, 0, None) != 0 and b"activation" in lib.nphm_last_error()
    assert lib.nphm_layer16_backward(16, 16, 16, None, 16, 16, None, 4, 4, 4, 1, 2, 1.0, 16, 1 << 30, None) != 0 and b"null" in lib.nphm_last_error()
    assert lib.nphm_layer16_backward(16, 16, 16, 16, 16, 16, None, 4, 4, 4, 1, 2, 1.0, 16, 0, None) != 0 and b"workspace" in lib.nphm_last_error()

    def clip(ins, outs, counts, dtypes):
        n = len(ins)
        return lib.nphm_clip_grads((ctypes.c_void_p * n)(*ins), (ctypes.c_void_p * n)(*outs), (ctypes.c_int64 * n)(*counts),
                                   (ctypes.c_int * n)(*dtypes), n, 0, 1.0, 16, 16, 0, None)
    big = 1 << 20
    assert clip([big, big + 100], [big, big + 100], [64, 64], [1, 1]) != 0 and b"share memory" in lib.nphm_last_error()
    assert clip([big, big], [big, big], [64, 64], [1, 1]) != 0 and b"share memory" in lib.nphm_last_error()          # the same twice
    assert clip([big], [big + 16], [64], [1]) != 0 and b"share memory" in lib.nphm_last_error()                       # shifted by a few
    assert clip([big, 2 * big], [2 * big, 3 * big], [64, 64], [1, 1]) != 0 and b"share memory" in lib.nphm_last_error()
    assert clip([big, big], [2 * big, 3 * big], [64, 64], [1, 1]) != 0 and b"workspace" in lib.nphm_last_error()     # read twice: fine
    assert clip([big], [big], [-1], [1]) != 0 and b"count" in lib.nphm_last_error()
    assert clip([big], [big], [1], [7]) != 0 and b"dtype" in lib.nphm_last_error()


def test_build_notices_another_pytorch_and_makes_the_c_library_first(tmp_path, monkeypatch):
    """with compilers that only write their output's name down: nothing of the tree is touched"""
    import subprocess
    from nphm_amd import build as B
    for name, path in (("OUT", "a.so"), ("TORCH_OUT", "b.so"), ("STAMP", "s.stamp"), ("OBJ_CACHE", "cache")):
        monkeypatch.setattr(B, name, str(tmp_path / path))
    made, broken = [], []

    def run(cmd, **kw):
        if "-o" in cmd:
            if broken and broken[0] in cmd[cmd.index("-o") + 1]:
                raise subprocess.CalledProcessError(1, cmd)
            made.append(cmd[cmd.index("-o") + 1])
            open(made[-1], "w").close()
        return subprocess.CompletedProcess(cmd, 0, b"", b"")

    class Popen:
        def __init__(self, cmd, **kw):
            run(cmd)

        def wait(self):
            return 0

    monkeypatch.setattr(B.subprocess, "run", run)
    monkeypatch.setattr(B.subprocess, "Popen", Popen)
    broken.append("torch_ops")
    assert B._stale()
    with pytest.raises(subprocess.CalledProcessError):
        B.build()
    assert (tmp_path / "a.so").exists() and not (tmp_path / "b.so").exists() and B._stale()
    broken.clear()
    B.build()
    assert (tmp_path / "b.so").exists() and not B._stale()
    made.clear()
    B.build()
    assert not made
    monkeypatch.setattr(B, "version", lambda name: "0.0")            # another PyTorch: its side is made again, with time stamps as they were
    assert B._stale()
    B.build()
    assert any("b.so" in m for m in made) and not B._stale()
    monkeypatch.setattr(B, "FLAGS", B.FLAGS + ["-g"])
    assert B._stale()

    def unknown(name):
        raise B.PackageNotFoundError(name)

    monkeypatch.setattr(B, "version", unknown)
    B.build()                                                        # a PyTorch without package data is no reason to fail
    assert not B._stale()


# ---- rows of a table ------------------------------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    return torch.device("cuda:0")


ROW_CASES = [(1, 1, 1), (7, 3, 5), (24, 1344, 16), (1000, 64, 257), (50, 200, 1), (333, 1001, 300), (4099, 40, 2500), (9, 515, 10000),
             (70001, 24, 9001), (3, 8, 40000), (2000, 2048, 700),
             (3000, 5000, 10), (3000, 20000, 7), (300000, 8, 256), (5000, 100, 200), (2, 9000, 256)]


@gpu
@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("V,D,N", ROW_CASES)
def test_lookup_and_gradient(dev, t, V, D, N):
    gen = torch.Generator().manual_seed(V * 31 + D + N)
    table = torch.randn(V, D, generator=gen).to(t).to(dev)
    idx = (torch.rand(N, generator=gen) ** 3 * V).long().clamp_(0, V - 1).to(dev)
    for kind in (torch.int64, torch.int32):
        for s in (1.0, 0.37):
            got = T.lookup_rows(table, idx.to(kind), scale=s)
            want = table.double()[idx] * s
            s32 = float(np.float32(s))
            assert got.dtype == t and got.shape == (N, D)
            within(got, want, want.abs() * (half_step(t) + 2 * F32 + abs(s32 - s) / s) + tiny(t))
    if True:
        g = torch.randn(N, D, generator=gen).to(t).to(dev)
        pad = int(idx[0])
        for padding in (None, pad):
            got = T.lookup_rows_grad(g, idx, V, scale=0.37, padding_idx=padding)
            keep = torch.ones(N, dtype=torch.bool, device=dev) if padding is None else idx != padding
            want = torch.zeros(V, D, dtype=torch.float64, device=dev).index_put_((idx[keep],), g[keep].double(), accumulate=True) * 0.37
            mag = torch.zeros(V, D, dtype=torch.float64, device=dev).index_put_((idx[keep],), g[keep].double().abs(), accumulate=True) * 0.37
            many = torch.bincount(idx[keep], minlength=V)[:, None].double()
            within(got, want, mag * (many + 2) * F32 + want.abs() * (half_step(t) + F32) + tiny(t))
            assert torch.equal(got, T.lookup_rows_grad(g, idx.int(), V, scale=0.37, padding_idx=padding))      # bits


@gpu
@pytest.mark.parametrize("t", FLOATS)
def test_rows_strides_shapes_and_alignment(dev, t):
    gen = torch.Generator().manual_seed(5)
    wide = torch.randn(40, 77, generator=gen).to(t).to(dev)
    idx = torch.randint(0, 40, (3, 1, 4), generator=gen).to(dev)
    for table in (wide[:, 3:70], wide[:, ::2], wide.t(), wide[::3], wide[:1].expand(40, 77), wide.reshape(-1)[1:1 + 40 * 70].view(40, 70)):
        i = idx % table.shape[0]
        got = T.lookup_rows(table, i)
        assert torch.equal(got, table[i])
        every_second = i.reshape(-1).repeat(2)[::2]
        assert torch.equal(T.lookup_rows(table, every_second), table[every_second])
    g = torch.randn(12, 77, generator=gen).to(t).to(dev)
    for grad in (g, g[:, 1:70], g.t().contiguous().t(), g[:1].expand(12, 77)):
        got = T.lookup_rows_grad(grad.reshape(3, 1, 4, -1), idx, 40)
        assert torch.equal(got, T.lookup_rows_grad(grad.contiguous(), idx.reshape(-1), 40))
    assert T.lookup_rows(wide, torch.empty(0, 2, dtype=torch.long, device=dev)).shape == (0, 2, 77)
    assert not T.lookup_rows_grad(g[:0], torch.empty(0, dtype=torch.long, device=dev), 11).any()
    assert torch.equal(T.lookup_rows(wide, torch.tensor(4, device=dev)), wide[4])


@gpu
@pytest.mark.parametrize("N", [20, 900, 20000])
def test_indices_outside_the_table(dev, N):
    """rows of NaN, no gradient, nothing read or written beside the table (rows around it stay)"""
    V, D = 30, 72
    around = torch.randn(V + 20, D, device=dev)
    table = around[10:10 + V]
    idx = torch.arange(N, device=dev) % V
    idx[3], idx[7], idx[11], idx[12] = -1, V, 2 ** 40, -2 ** 62
    bad = (idx < 0) | (idx >= V)
    got = T.lookup_rows(table, idx)
    assert bool(got[bad].isnan().all()) and torch.equal(got[~bad], table[idx[~bad]])
    g = torch.randn(N, D, device=dev)
    assert torch.equal(T.lookup_rows_grad(g, idx, V), T.lookup_rows_grad(g[~bad], idx[~bad], V))
    assert not T.lookup_rows_grad(g, torch.full((N,), -5, device=dev), V).any()
    before = around.clone()
    T.renorm_rows_(table, idx, 0.5)
    assert torch.equal(around[:10], before[:10]) and torch.equal(around[10 + V:], before[10 + V:])


@gpu
@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("V,D,N", [(1, 1, 1), (7, 3, 5), (24, 1344, 16), (50, 61, 300), (4099, 130, 9001), (6, 20000, 3)])
def test_sparse_gradient_has_an_entry_for_every_index(dev, t, V, D, N):
    """in the order of the indices, one rounding of scale * g each; padding and indices outside the table: row 0 and zeros, NaN or not"""
    gen = torch.Generator().manual_seed(V + D + N)
    table = torch.randn(V, D, generator=gen).to(t).to(dev).requires_grad_()
    wide = torch.randn(N, D + 3, generator=gen).to(t).to(dev)
    idx = torch.randint(-1, V + 1, (N,), generator=gen).to(dev)
    padding = V // 2
    kept = (idx >= 0) & (idx < V) & (idx != padding)
    for kind in (torch.int64, torch.int32):
        for g in (wide[:, :D].contiguous(), wide[:, 2:D + 2], wide[:1, :D].expand(N, D), wide[:, :D].index_fill(0, (~kept).nonzero()[:, 0], math.nan)):
            grad, = torch.autograd.grad(T.lookup_rows(table, idx.to(kind), 0.37, padding_idx=padding, sparse=True), table, g)
            assert grad.is_sparse and grad.dtype == t and grad.shape == (V, D) and grad._indices().dtype == torch.int64
            assert torch.equal(grad._indices()[0], torch.where(kept, idx, 0))
            assert not grad._values()[~kept].any()
            want = g[kept].double() * 0.37
            within(grad._values()[kept], want, want.abs() * (half_step(t) + 3 * F32) + tiny(t))
    grad, = torch.autograd.grad(T.lookup_rows(table, idx[:0].reshape(0, 2), sparse=True), table, wide[:0, :D].reshape(0, 2, D))
    assert grad.is_sparse and grad._nnz() == 0 and not grad.to_dense().any()


@gpu
@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("V,D,N", [(9, 600, 9000), (700, 515, 9001), (20011, 640, 9000), (60000, 512, 8193), (5000, 5001, 10000)])
def test_long_rows_named_by_many_indices(dev, t, V, D, N):
    """one call after another on the memory that the call before left: rows that nobody names are zeros, padding and foreign indices too"""
    gen = torch.Generator().manual_seed(V + D + N)
    g = torch.randn(N, D, generator=gen).to(t).to(dev)
    for turn in range(3):
        idx = torch.randint(-2, V + 2, (N,), generator=gen)
        idx[: N // 3] = (idx[: N // 3] % max(1, V // 50)) * min(V, 49)        # some rows over and over, and rows that nobody names
        idx = idx.clamp(max=V + 1).to(dev)
        padding = None if turn == 0 else V // 2
        keep = (idx >= 0) & (idx < V) & (idx != (-7 if padding is None else padding))
        got = T.lookup_rows_grad(g, idx.int() if turn == 2 else idx, V, padding_idx=padding)
        want = torch.zeros(V, D, dtype=torch.float64, device=dev).index_put_((idx[keep],), g[keep].double(), accumulate=True)
        mag = torch.zeros(V, D, dtype=torch.float64, device=dev).index_put_((idx[keep],), g[keep].double().abs(), accumulate=True)
        many = torch.bincount(idx[keep], minlength=V)[:, None].double()
        within(got, want, mag * (many + 2) * F32 + want.abs() * (half_step(t) + F32) + tiny(t))
        assert not got[many[:, 0] == 0].any()


@gpu
def test_rows_that_fill_the_last_cache(dev):
    """the ways through memory that only large calls take (results above 256 MiB, odd rows), for every number of indices; whole numbers, so
    that any order of sums is exact"""
    V, D = 17000, 4099
    gen = torch.Generator(device=dev).manual_seed(8)
    table = torch.randint(-8, 9, (V, D), device=dev, generator=gen).float()
    for N in (9000, V, V + 1):
        idx = torch.randint(0, V, (N,), device=dev, generator=gen)
        assert torch.equal(T.lookup_rows(table, idx), table.index_select(0, idx))
    for N in (200, 4000, 9000):
        idx = torch.randint(0, V, (N,), device=dev, generator=gen)
        idx[N // 2:] %= 40
        got = T.lookup_rows_grad(table[:N], idx, V)
        assert torch.equal(got, torch.zeros(V, D, device=dev).index_add_(0, idx, table[:N]))
        del got


@gpu
def test_row_gradients_do_not_overflow_in_sums(dev):
    """fp16 rows whose partial sums leave the type's range and come back"""
    g = torch.full((2000, 24), 60000.0, dtype=torch.float16, device=dev)
    g[1000:] = -60000.0
    got = T.lookup_rows_grad(g, torch.zeros(2000, dtype=torch.long, device=dev), 2)
    assert torch.equal(got, torch.zeros_like(got))
    g[5] = math.nan
    assert bool(T.lookup_rows_grad(g, torch.zeros(2000, dtype=torch.long, device=dev), 2)[0].isnan().all())
    assert not T.lookup_rows_grad(g, torch.zeros(2000, dtype=torch.long, device=dev), 2, padding_idx=0).any()      # NaN in a padded place


@gpu
def test_row_offsets_behind_32_bits(dev):
    """a table of 1.2e9 values (4.9 GB): rows at its end, and a gradient of its size"""
    V, D = 1200001, 1024
    table = torch.empty(V, D, device=dev)
    idx = torch.tensor([V - 1, 0, V - 1, 1048576, V - 2, 524288, 2097151 % V], device=dev).repeat(60)
    table[idx] = torch.randn(len(idx), D, device=dev)
    assert torch.equal(T.lookup_rows(table, idx), table[idx])
    g = torch.randn(len(idx), D, device=dev)
    for n in (7, len(idx)):
        got = T.lookup_rows_grad(g[:n], idx[:n], V)
        want = torch.zeros(V, D, device=dev, dtype=torch.float64).index_put_((idx[:n],), g[:n].double(), accumulate=True)
        named = torch.unique(idx[:n])
        within(got[named], want[named], want[named].abs() * F32 + n * F32 * g[:n].abs().max().double() * n / 3)
        assert int((got != 0).any(1).sum()) == len(named)
        del got, want
    T.renorm_rows_(table, idx, 1.0)
    assert float(table[idx].norm(dim=1).max()) <= 1 + 1e-6


@gpu
@pytest.mark.parametrize("t", FLOATS)
def test_renorm_scales_named_rows_once(dev, t):
    table = (torch.randn(60, 300, generator=torch.Generator().manual_seed(2)) * torch.linspace(0.01, 0.2, 60)[:, None]).to(t).to(dev)
    idx = torch.tensor([5, 5, 59, 40, 40, 40, 0, 30], device=dev)
    before, version = table.clone(), table._version
    T.renorm_rows_(table, idx, 1.0)
    assert table._version > version
    want = before.double()
    for v in set(idx.tolist()):
        n = float(want[v].norm())
        if n > 1.0:
            want[v] *= 1.0 / (n + 1e-7)
    within(table, want, want.abs() * (half_step(t) + 2 * F32) + tiny(t))
    untouched = [v for v in range(60) if v not in idx.tolist()]
    assert torch.equal(table[untouched], before[untouched])
    ref = torch.nn.functional.embedding(idx, before.float().clone(), max_norm=1.0)
    assert float((T.lookup_rows(table, idx).float() - ref).abs().max()) <= float(ref.abs().max()) * (half_step(t) + 4e-7)


@gpu
def test_latent_codes_module_against_embedding(dev):
    for sparse in (False, True):
        for padding in (None, 2):
            ours = T.LatentCodes(12, 40, padding_idx=padding, max_norm=0.9, sparse=sparse, scale=1.5, device=dev)
            ref = torch.nn.Embedding(12, 40, padding_idx=padding, max_norm=0.9, sparse=sparse).to(dev)
            ref.load_state_dict(ours.state_dict())
            idx = torch.tensor([[1, 2, 1], [11, 2, 0]], device=dev)
            a, b = ours(idx), ref(idx) * 1.5
            go = torch.randn_like(a)
            a.backward(go)
            b.backward(go)
            ga, gb = [m.weight.grad.to_dense() if sparse else m.weight.grad for m in (ours, ref)]
            assert ours.weight.grad.is_sparse == sparse
            assert float((a - b).detach().abs().max()) <= 1e-6 and float((ga - gb).abs().max()) <= 2e-6 * float(gb.abs().max())
            assert float((ours.weight - ref.weight).detach().abs().max()) <= 4 * F32
            if sparse:       # both kinds step the trainer's optimiser
                torch.optim.SparseAdam([ours.weight], lr=1e-3).step()


# ---- dense layer ----------------------------------------------------------------------------------------------------------------

def layer_inputs(dev, t, M, N, K, bias, residual, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed + M + 3 * N + 7 * K)
    r = lambda *s: torch.randn(*s, device=dev, generator=gen)  # noqa: E731
    return (r(M, K).to(t), (r(N, K) / math.sqrt(K)).to(t), (0.1 * r(N)).to(t) if bias else None, r(M, N).to(t) if residual else None,
            r(M, N).to(t))


def act64(z, act, beta):
    """value and slope, from their formulas"""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    if act == "gelu":
        c = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return torch.logaddexp(z * beta, torch.zeros_like(z)) / beta, torch.sigmoid(z * beta)


CURVE = {"none": 0.0, "relu": 0.0, "silu": 0.5, "gelu": 0.8}          # largest |a''|; Softplus: beta / 4


def check_layer(dev, t, M, N, K, act, beta=1.0, bias=True, residual=False, seed=0):
    x, w, b, r, g = layer_inputs(dev, t, M, N, K, bias, residual, seed)
    leaves = [v.clone().requires_grad_() if v is not None else None for v in (x, w, b, r)]
    y = T.linear_act(leaves[0], leaves[1], leaves[2], activation=act, beta=beta, residual=leaves[3])
    y.backward(g)
    plain = T.linear_act(x, w, b, activation=act, beta=beta, residual=r)
    assert torch.equal(plain, y.detach()) and not plain.requires_grad
    h = half_step(t)
    xd, wd, gd = x.double(), w.double(), g.double()
    z = xd @ wd.t()
    mag = xd.abs() @ wd.abs().t()
    if bias:
        z, mag = z + b.double(), mag + b.double().abs()
    ez = (K + 4) * 2 * F32 * mag
    a, slope = act64(z, act, beta)
    want = a + (r.double() if residual else 0)
    # a: slope at most 1.13; exp, log and erf to 2^-20 of what enters them; Softplus above 20 / beta is z: off by exp(-20) / beta
    ey = 1.13 * ez + 2.0 ** -20 * (a.abs() + z.abs()) + (2.1e-9 / beta if act == "softplus" else 0) + F32 * want.abs()
    within(y.detach(), want, ey + h * (want.abs() + ey) + tiny(t))
    # gz: z is kept with one rounding, |z a''(z)| <= 0.5 for every activation; then gz is rounded once itself
    curve = beta / 4 if act == "softplus" else CURVE[act]
    gz = gd * slope
    dz = gd.abs() * ((0.55 * h if act not in ("none", "relu") else 0) + curve * ez + 2.0 ** -19)
    if act == "relu":
        dz = dz + gd.abs() * (z.abs() <= ez + tiny(t))
    rounded = dz + (h * (gz.abs() + dz) + tiny(t) if act != "none" else 0)
    wants = [(gz @ wd, rounded @ wd.abs() + (N + 4) * 2 * F32 * ((gz.abs() + rounded) @ wd.abs())),
             (gz.t() @ xd, rounded.t() @ xd.abs() + (M + 4) * 2 * F32 * ((gz.abs() + rounded).t() @ xd.abs())),
             (gz.sum(0), dz.sum(0) + (M + 4) * F32 * (gz.abs() + dz).sum(0))]
    for leaf, (v, e) in zip(leaves[:3], wants):
        if leaf is not None:
            assert leaf.grad.dtype == t
            within(leaf.grad, v, e + h * (v.abs() + e) + tiny(t))
    if residual:
        assert torch.equal(leaves[3].grad, g)
    return leaves, y


@gpu
@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("act,beta", [("none", 1.0), ("relu", 1.0), ("silu", 1.0), ("gelu", 1.0), ("softplus", 1.0), ("softplus", 100.0)])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (5, 130, 515), (70, 64, 64), (300, 257, 200)])
def test_layer_and_gradients(dev, t, act, beta, M, N, K):
    check_layer(dev, t, M, N, K, act, beta, bias=True, residual=M != 70)


@gpu
@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("M,N,K", [(1, 1024, 512), (16, 333, 4096), (17, 40, 1000), (33, 2048, 96), (64, 3, 512), (129, 1, 8), (128, 128, 128), (256, 256, 256),
                                   (257, 513, 129), (1000, 512, 512), (4095, 96, 515), (2, 5000, 24), (3000, 8, 1344), (515, 1030, 1032),
                                   (20000, 64, 72), (9, 70, 30000), (70000, 40, 72), (40000, 200, 130), (17000, 513, 300)])
@pytest.mark.parametrize("bias,residual", [(True, False), (False, True)])
def test_layer_sizes(dev, t, M, N, K, bias, residual):
    check_layer(dev, t, M, N, K, "softplus" if residual else "none", 20.0, bias=bias, residual=residual)


@gpu
def test_layer_strides_shapes_and_refusals(dev):
    t = torch.bfloat16
    x, w, b, r, g = layer_inputs(dev, t, 60, 48, 40, True, True)
    want = T.linear_act(x, w, b, "gelu", residual=r)
    wide = torch.zeros(60, 100, dtype=t, device=dev)
    wide[:, 7:47] = x
    spread = torch.zeros(48, 80, dtype=t, device=dev)
    spread[:, ::2] = w
    packed = torch.zeros(60 * 48 + 1, dtype=t, device=dev)
    packed[1:] = r.reshape(-1)
    for args in ((wide[:, 7:47], w, b, r), (x, w.t().contiguous().t(), b, r), (x, spread[:, ::2], b, r), (x, w, b, r.t().contiguous().t()),
                 (x, w, b, packed[1:].view(60, 48)), (x, w, b.repeat_interleave(2)[::2], r)):
        assert torch.equal(T.linear_act(*args[:3], "gelu", residual=args[3]), want)
    batched = T.linear_act(x.view(3, 4, 5, 40), w, b, "gelu", residual=r.view(3, 4, 5, 48))
    assert torch.equal(batched.view(60, 48), want)
    assert torch.equal(T.linear_act(x[0], w, b, "gelu", residual=r[0]).view(1, 48), T.linear_act(x[:1], w, b, "gelu", residual=r[:1]))
    empty = x[:0].clone().requires_grad_()
    w2 = w.clone().requires_grad_()
    T.linear_act(empty, w2, b).sum().backward()
    assert empty.grad.shape == (0, 40) and not w2.grad.any()
    # a gradient that is one value spread over the result
    x2, w2 = x.clone().requires_grad_(), w.clone().requires_grad_()
    T.linear_act(x2, w2, b, "silu").sum().backward()
    x3, w3 = x.clone().requires_grad_(), w.clone().requires_grad_()
    T.linear_act(x3, w3, b, "silu").backward(torch.ones(60, 48, dtype=t, device=dev))
    assert torch.equal(x2.grad, x3.grad) and torch.equal(w2.grad, w3.grad)
    for bad in (dict(activation="tanh"), dict(activation="softplus", beta=0.0), dict(residual=r[0]), dict(residual=r.float()), dict(bias=b[:-1]),
                dict(bias=b.half())):
        with pytest.raises((ValueError, TypeError)):
            T.linear_act(x, w, **bad)
    for pair in ((x.float(), w.float()), (x, w[:, :-1]), (x, w.half()), (x, w.cpu())):
        with pytest.raises((ValueError, TypeError)):
            T.linear_act(*pair)
    # second order is refused, not wrong
    x4 = x.clone().requires_grad_()
    (gx,) = torch.autograd.grad(T.linear_act(x4, w, b, "silu").sum(), x4, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


@gpu
@pytest.mark.parametrize("t", HALVES)
def test_layer_gradient_against_differences(dev, t):
    """the directional derivative of sum(y go) along d, by central differences of the 64-bit formula at the layer's own inputs; the layer's
    dot product with its gradients is off by their bounds (checked entry by entry above): 4 roundings of t of the magnitudes"""
    x, w, b, _, go = layer_inputs(dev, t, 40, 33, 24, True, False, seed=3)
    leaves = [v.clone().requires_grad_() for v in (x, w, b)]
    T.linear_act(*leaves, "gelu").backward(go)

    def f(xx, ww, bb):
        return (act64(xx @ ww.t() + bb, "gelu", 1.0)[0] * go.double()).sum()
    gen = torch.Generator(device=dev).manual_seed(9)
    for k in range(3):
        d = torch.randn(leaves[k].shape, device=dev, generator=gen).double()
        args = [v.double() for v in (x, w, b)]
        up, down = list(args), list(args)
        up[k], down[k] = args[k] + 1e-4 * d, args[k] - 1e-4 * d
        numeric = float(f(*up) - f(*down)) / 2e-4
        own = float((leaves[k].grad.double() * d).sum())
        z = x.double() @ w.double().t() + b.double()
        gz = (go.double() * act64(z, "gelu", 1.0)[1]).abs()
        span = [gz @ w.double().abs(), gz.t() @ x.double().abs(), gz.sum(0)][k]
        assert abs(own - numeric) <= 4 * half_step(t) * float((span * d.abs()).sum()) + 1e-5


@gpu
def test_layer_special_values(dev):
    """NaN and infinities stay in their rows; large values do not leave a gradient that is no number"""
    t = torch.float16
    x, w, b, _, g = layer_inputs(dev, t, 200, 96, 64, True, False)
    want = T.linear_act(x, w, b, "gelu")
    x[17, 3], x[130, 5] = math.nan, math.inf
    got = T.linear_act(x, w, b, "gelu")
    rows = torch.ones(200, dtype=torch.bool, device=dev)
    rows[17] = rows[130] = False
    assert torch.equal(got[rows], want[rows]) and bool(got[17].isnan().all()) and not bool(torch.isfinite(got[130]).all())
    big = torch.full((8, 64), 6000.0, dtype=t, device=dev, requires_grad=True)
    one = torch.ones(16, 64, dtype=t, device=dev)
    for act in ("silu", "gelu", "softplus", "relu"):
        big.grad = None
        T.linear_act(big, one, None, act).backward(torch.ones(8, 16, dtype=t, device=dev))      # z = 384 000: above the type's range
        assert torch.equal(big.grad, torch.full_like(big, 16.0)), act
    for act in ("silu", "gelu", "softplus", "relu"):
        big.grad = None
        T.linear_act(big, -one, None, act).backward(torch.ones(8, 16, dtype=t, device=dev))
        assert not big.grad.any(), act


@gpu
def test_layer_gradients_asked_one_by_one(dev):
    """whatever subset of the four gradients is asked for, each has the same bits"""
    x, w, b, r, g = layer_inputs(dev, torch.bfloat16, 200, 72, 130, True, True)
    full = [v.clone().requires_grad_() for v in (x, w, b, r)]
    T.linear_act(*full[:3], "silu", residual=full[3]).backward(g)
    for mask in range(1, 16):
        leaves = [v.clone().requires_grad_(bool(mask >> k & 1)) for k, v in enumerate((x, w, b, r))]
        T.linear_act(*leaves[:3], "silu", residual=leaves[3]).backward(g)
        for k, (leaf, ref) in enumerate(zip(leaves, full)):
            assert (leaf.grad is None) == (not mask >> k & 1)
            assert leaf.grad is None or torch.equal(leaf.grad, ref.grad)


@gpu
def test_saved_tensors_that_change_are_noticed(dev):
    x, w, b, _, g = layer_inputs(dev, torch.bfloat16, 20, 16, 24, True, False)
    w.requires_grad_()
    y = T.linear_act(x, w, b, "gelu")
    x.zero_()
    with pytest.raises(RuntimeError):
        y.backward(g)
    table, idx = torch.randn(5, 8, device=dev, requires_grad=True), torch.tensor([1, 2], device=dev)
    rows = T.lookup_rows(table, idx)
    idx.add_(1)
    with pytest.raises(RuntimeError):
        rows.sum().backward()


@gpu
def test_inference_mode(dev):
    with torch.inference_mode():
        x, w, b, r, _ = layer_inputs(dev, torch.bfloat16, 20, 16, 24, True, True)
        g = [torch.randn(100, device=dev), torch.randn(7, device=dev)]
        table, idx = torch.randn(5, 8, device=dev), torch.tensor([1, 2], device=dev)
        assert T.linear_act(x, w, b, "gelu", residual=r).shape == (20, 16)
        T.clip_grads(g, 0.1)
        assert abs(float(T.grad_norm(g)) - 0.1) <= 1e-6
        T.renorm_rows_(table, idx, 0.5)
        assert float(T.lookup_rows(table, idx).norm(dim=1).max()) <= 0.5 * (1 + 4 * F32)


@gpu
def test_layer_offsets_behind_32_bits(dev):
    """a result of 2.3e9 values (4.6 GB) and its gradients: spot checks in the last rows against 64 bits, and the whole-sum gradients"""
    t, M, N, K = torch.bfloat16, 70000, 32768, 64
    x, w, b, _, _ = layer_inputs(dev, t, M, N, K, True, False)
    leaves = [v.requires_grad_() for v in (x, w, b)]
    y = T.linear_act(*leaves, "relu")
    at = torch.tensor([0, 1, 40000, 65536, M - 2, M - 1], device=dev)
    xd, wd, bd = x.detach().double(), w.detach().double(), b.detach().double()
    z = xd[at] @ wd.t() + bd
    ez = (K + 4) * 2 * F32 * (xd[at].abs() @ wd.abs().t() + bd.abs())
    within(y.detach()[at], z.clamp(min=0), ez + half_step(t) * (z.abs() + ez) + tiny(t))
    go = torch.zeros(M, N, dtype=t, device=dev)
    go[at] = torch.randn(len(at), N, device=dev).to(t)
    y.backward(go)
    live = (z > 0) & (z.abs() > ez)
    edge = (z.abs() <= ez).double() * go[at].double().abs()
    gz = go[at].double() * live
    # e: what a gradient is off before it is rounded (an entry whose z lies within its own error of 0 counts on one side and not on the other);
    # the rounding is then one of |gradient| + e, not of |gradient|: 1.002 of the bound was seen without it, at an entry with |ref| 0.05, e 2.09
    h = half_step(t)

    def bound(ref, e):
        return e + h * (ref.abs() + e) + tiny(t)
    ref = gz @ wd
    within(x.grad[at], ref, bound(ref, edge @ wd.abs() + (N + 4) * 2 * F32 * (gz.abs() @ wd.abs())))
    rest = torch.ones(M, dtype=torch.bool, device=dev)
    rest[at] = False
    assert not x.grad[rest].any()
    ref = gz.t() @ xd[at]
    within(w.grad, ref, bound(ref, edge.t() @ xd[at].abs() + 16 * F32 * (gz.abs().t() @ xd[at].abs())))
    within(b.grad, gz.sum(0), bound(gz.sum(0), edge.sum(0) + 16 * F32 * gz.abs().sum(0)))


@gpu
def test_layer_with_more_rows_than_a_grid_axis(dev):
    """2^21 + 3 rows: more tiles of rows than one axis of a launch may have blocks"""
    t, M, N, K = torch.float16, (1 << 21) + 3, 8, 8
    x, w, b, _, g = layer_inputs(dev, t, M, N, K, True, False)
    leaves = [v.requires_grad_() for v in (x, w, b)]
    y = T.linear_act(*leaves, "silu")
    y.backward(g)
    z = x.detach().double() @ w.detach().double().t() + b.detach().double()
    a, slope = act64(z, "silu", 1.0)
    gz = g.double() * slope
    want = gz.sum(0)
    # fp32 sums over M entries in tiles: at most tile height + tiles adds follow one another, 2^14 here
    dz = g.double().abs() * (0.55 * half_step(t) + 2.0 ** -19 + 0.5 * 24 * F32 * (1 + z.abs()))
    within(b.grad, want, dz.sum(0) + 2 ** 14 * F32 * gz.abs().sum(0) + half_step(t) * want.abs())
    within(y.detach()[-5:], a[-5:], half_step(t) * a[-5:].abs() + 1e-5)
    within(x.grad[-5:], gz[-5:] @ w.detach().double(), (dz[-5:] + half_step(t) * gz[-5:].abs()) @ w.detach().double().abs() * 1.01
           + half_step(t) * (gz[-5:] @ w.detach().double()).abs() + tiny(t))


@gpu
@pytest.mark.parametrize("t", ["bf16", "fp16"])
def test_decoder_trains_with_16_bit_hidden_layers(dev, t):
    """DeepSDF.train_precision: the same bits as the layers called one by one, and the fp32 tier untouched by it"""
    torch.manual_seed(0)
    net = DeepSDF(lat_dim=32, hidden_dim=128, nlayers=6, beta=100, out_dim=1).to(dev).train()
    xyz = torch.randn(2, 300, 3, device=dev) * 0.3
    lat = (torch.randn(2, 1, 32, device=dev) * 0.1).requires_grad_()
    before = net.evaluate_train_hip(xyz, lat)
    net.train_precision = t
    out = net.evaluate_train_hip(xyz, lat)
    out.square().sum().backward()
    grads = [p.grad.clone() for p in net.parameters()] + [lat.grad.clone()]
    net.zero_grad()
    lat.grad = None
    h = {"bf16": torch.bfloat16, "fp16": torch.float16}[t]
    inp = torch.cat([xyz, lat.expand(2, 300, 32)], -1).reshape(600, -1)
    x = inp
    for k in range(6):
        lin = getattr(net, f"lin{k}")
        if k == 0:
            x = _DenseLayerFn.apply(x, lin.weight, lin.bias, 1.0, 100.0)
        elif k == 3:
            x = _DenseLayerFn.apply(torch.cat([x.float(), inp], -1), lin.weight, lin.bias, 1 / math.sqrt(2), 100.0)
        else:
            x = T.linear_act(x.to(h), lin.weight.to(h), lin.bias.to(h), "softplus", 100.0)
    want = torch.nn.functional.linear(x.float(), net.lin6.weight, net.lin6.bias).view(2, 300, 1)
    assert torch.equal(out, want)
    want.square().sum().backward()
    for a, p in zip(grads, list(net.parameters()) + [lat]):
        assert torch.equal(a, p.grad)
    net.train_precision = "fp32"
    assert torch.equal(net.evaluate_train_hip(xyz, lat), before)
    net.train_precision = "fp8"
    with pytest.raises(ValueError):
        net.evaluate_train_hip(xyz, lat)


@gpu
@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("rows", [600, 20000])
def test_small_gradients_come_through_16_bit_layers(dev, t, rows):
    """a loss of 2^-k times the size (a mean over points, a small weight) gives 2^-k times the gradients.  At their own size fp16 would hold the
    smaller ones as zero.  Both passes round to 16 bits alike but for entries near fp16's smallest, off by half of 2^-24 where the
    largest is 2^10 over the number of rows: a rounding of the gradient's 2-norm covers them, a few bits lost do not pass."""
    torch.manual_seed(0)
    net = DeepSDF(lat_dim=32, hidden_dim=128, nlayers=6, beta=100, out_dim=1).to(dev).train()
    net.train_precision = t
    xyz = torch.randn(1, rows, 3, device=dev) * 0.3
    lat = (torch.randn(1, 1, 32, device=dev) * 0.1).requires_grad_()
    go = torch.randn(1, rows, 1, device=dev)
    leaves = [lat, *net.parameters()]
    want = torch.autograd.grad(net.evaluate_train_hip(xyz, lat), leaves, go)
    assert all(bool(torch.isfinite(g).all()) and float(g.abs().max()) > 0 for g in want)
    for k in (12, 24, 60):
        got = torch.autograd.grad(net.evaluate_train_hip(xyz, lat), leaves, go * 2.0 ** -k)
        for a, b in zip(got, want):
            assert float((a.double() * 2.0 ** k - b.double()).norm()) <= half_step(torch.float16) * float(b.double().norm()), k
    zero = torch.autograd.grad(net.evaluate_train_hip(xyz, lat), leaves, go * 0)
    assert not any(bool(g.any()) for g in zero)
    net.lin1.weight.requires_grad_(False)                            # frozen parameters: none for them, the same for the others
    net.lin4.bias.requires_grad_(False)
    some = [p for p in leaves if p.requires_grad]
    got = torch.autograd.grad(net.evaluate_train_hip(xyz, lat), some, go)
    assert all(torch.equal(a, b) for a, b in zip(got, [g for g, p in zip(want, leaves) if p.requires_grad]))
    for p in net.parameters():
        p.requires_grad_(False)
    assert torch.equal(torch.autograd.grad(net.evaluate_train_hip(xyz, lat), lat, go)[0], want[0])
    net.requires_grad_(True)
    go[0, 5] = math.inf                                              # shows, and is not scaled away
    assert not all(bool(torch.isfinite(g).all()) for g in torch.autograd.grad(net.evaluate_train_hip(xyz, lat), leaves, go * 2.0 ** -24))


def test_backward_workspace_is_for_the_operands_handed_over():
    """no x: no gradient of the weight, no weight: none of x - and no room for what they would need (host arithmetic, no GPU)"""
    from nphm_amd import _lib
    lib = _lib.load()
    for M, N, K in ((4095, 1024, 515), (128, 128, 100000), (1, 4096, 4096), (100000, 128, 128), (3, 7, 5)):
        for act in (0, 4):
            full, x, w, none = [lib.nphm_layer16_backward_workspace_bytes(4096, *p, M, N, K, act) for p in ((4096, 4096), (4096, None), (None, 4096), (None, None))]
            assert none <= min(x, w) and max(x, w) <= full
            assert none < full or (N % 8 == 0 and K % 8 == 0 and act == 0 and full == x == w)      # (nothing but db's partial sums)


@gpu
@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("M,N,K", [(37, 64, 48), (130, 33, 21), (4095, 96, 515), (300, 512, 2000), (0, 8, 8)])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_only_the_gradients_that_are_asked_for(dev, t, M, N, K, act):
    """every choice of inputs that require one, and of those one pass asks for: the same bits as all of them together"""
    x, w, b, r, g = layer_inputs(dev, t, M, N, K, True, True)
    names = ("x", "weight", "bias", "residual")
    leaves = [v.clone().requires_grad_() for v in (x, w, b, r)]
    full = dict(zip(names, torch.autograd.grad(T.linear_act(*leaves[:3], act, residual=leaves[3]), leaves, g)))
    for need in range(1, 16):
        own = [v.clone().requires_grad_(bool(need >> i & 1)) for i, v in enumerate((x, w, b, r))]
        for ask in range(1, 16):
            if ask & ~need:
                continue
            picked = [i for i in range(4) if ask >> i & 1]
            got = torch.autograd.grad(T.linear_act(*own[:3], act, residual=own[3]), [own[i] for i in picked], g)
            for i, v in zip(picked, got):
                assert torch.equal(v, full[names[i]]), (need, ask, names[i])
    # no bias, no residual: the places of the others stay theirs
    two = [x.clone().requires_grad_(), r.clone().requires_grad_()]
    got = torch.autograd.grad(T.linear_act(two[0], w, None, act, residual=two[1]), two[1], g)
    assert torch.equal(got[0], g)
    got = torch.autograd.grad(T.linear_act(two[0], w, None, act, residual=two[1]), two[0], g)
    assert got[0].shape == x.shape


@gpu
def test_a_layer_keeps_what_its_gradients_read(dev):
    """a frozen weight's layer does not keep x (nor mind that it changes), frozen inputs' not the weight, the residual alone keeps nothing"""
    M, N, K = 1024, 512, 2048
    x, w, b, r, g = layer_inputs(dev, torch.bfloat16, M, N, K, True, True)
    leaf = x.clone().requires_grad_()
    want, = torch.autograd.grad(T.linear_act(leaf, w, b, "silu"), leaf, g)
    moving = leaf * 1
    y = T.linear_act(moving, w, b, "silu")
    moving.detach().zero_()                                          # (no gradient of the weight: x is not read again)
    got, = torch.autograd.grad(y, moving, g)
    assert torch.equal(got, want)
    weight = w.clone().requires_grad_()
    moving = weight * 1
    y = T.linear_act(x, moving, b, "silu")
    want, = torch.autograd.grad(T.linear_act(x, weight, b, "silu"), weight, g)
    moving.detach().zero_()
    got, = torch.autograd.grad(y, moving, g)
    assert torch.equal(got, want)
    residual = r.clone().requires_grad_()
    del y
    before = torch.cuda.memory_allocated()
    y = T.linear_act(x, w, b, "silu", residual=residual)
    assert torch.cuda.memory_allocated() - before == y.numel() * 2   # the result alone, no z beside it
    del y
    bias, free = b.clone().requires_grad_(), x.clone()
    before = torch.cuda.memory_allocated()
    y = T.linear_act(free, w, bias, "silu")
    del free
    assert torch.cuda.memory_allocated() - before == (2 * M * N - M * K) * 2         # y and z, and x has gone
    got, = torch.autograd.grad(y, bias, g)
    every = [v.clone().requires_grad_() for v in (x, w, b)]
    assert torch.equal(got, torch.autograd.grad(T.linear_act(*every, "silu"), every, g)[2])


# ---- gradient norm and clipping ---------------------------------------------------------------------------------------------------

def clip_bound(want, t):
    return want.abs() * (3 * F32 + (half_step(t) if t != torch.float32 else 0)) + tiny(t)


@gpu
@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("sizes", [[1], [0, 5, 0], [3, 1, 4, 1, 5, 9, 2, 6], [8192], [16385, 1], [70000, 3, 128, 40001], [1000] * 300, [2 ** 22 + 7]])
@pytest.mark.parametrize("limit", [0.1, 1e9])
def test_clip(dev, t, sizes, limit):
    gen = torch.Generator(device=dev).manual_seed(len(sizes) + sizes[0])
    grads = [(torch.randn(n, device=dev, generator=gen) * 0.5).to(t) for n in sizes]
    total = math.sqrt(math.fsum(float(g.double().square().sum()) for g in grads))
    most = max([float(g.abs().max()) for g in grads if g.numel()])
    assert abs(float(T.grad_norm(grads)) - total) <= total * 1.01 * F32
    assert float(T.grad_norm(grads, math.inf)) == most
    for kind, n in ((2.0, total), (math.inf, most)):
        out = [torch.full_like(g, 7.0) for g in grads]
        norm, got = T.clip_grads(grads, limit, norm_type=kind, out=out)
        assert abs(float(norm) - n) <= n * 1.01 * F32 and all(a is b for a, b in zip(got, out))
        f = min(1.0, limit / (n + 1e-6))
        for g, o in zip(grads, out):
            within(o, g.double() * f, clip_bound(g.double() * f, t))
        own = [g.clone() for g in grads]
        versions = [g._version for g in own]
        T.clip_grads(own, limit, norm_type=kind)
        assert all(torch.equal(a, b) for a, b in zip(own, out)) and all(g._version > v for g, v in zip(own, versions))


@gpu
def test_clip_mixed_types_views_and_layouts(dev):
    gen = torch.Generator(device=dev).manual_seed(1)
    flat = torch.randn(50000, device=dev, generator=gen)
    halves = torch.randn(50000, device=dev, generator=gen).half()
    base = [flat[1:4098], flat[5000:5007], halves[3:20003], torch.randn(40, 30, device=dev).bfloat16().t(), torch.randn(6, 50, device=dev)[:, ::5],
            torch.randn(3, 4, 5, device=dev).permute(2, 0, 1), torch.randn((), device=dev), halves[20003:20004]]
    total = math.sqrt(math.fsum(float(g.double().square().sum()) for g in base))
    want = [g.double() * min(1.0, 0.5 / (total + 1e-6)) for g in base]
    around = flat[4098:5000].clone(), halves[20004:].clone()
    out = [torch.empty(g.shape, dtype=g.dtype, device=dev) for g in base]
    T.clip_grads(base, 0.5, out=out)
    norm, _ = T.clip_grads(base, 0.5)
    assert abs(float(norm) - total) <= total * 1.01 * F32
    for g, o, w in zip(base, out, want):
        within(g, w, clip_bound(w, g.dtype))
        assert torch.equal(g, o)
    assert torch.equal(around[0], flat[4098:5000]) and torch.equal(around[1], halves[20004:])
    with pytest.raises(NphmAmdError):
        T.clip_grads([flat[:100], flat[50:150]], 1.0)
    with pytest.raises(NphmAmdError):
        T.clip_grads([flat[:100], flat[:100]], 1.0)
    with pytest.raises(TypeError):
        T.clip_grads([flat, flat.double()], 1.0)
    with pytest.raises(TypeError):
        T.clip_grads([flat, torch.zeros(3)], 1.0)
    with pytest.raises(ValueError):
        T.clip_grads([flat], 1.0, out=[flat[1:]])


@gpu
@pytest.mark.parametrize("value,kind", [(math.nan, 2.0), (math.nan, math.inf), (math.inf, 2.0), (-math.inf, math.inf)])
def test_clip_values_that_are_no_numbers_as_torch(dev, value, kind):
    def params():
        ps = [torch.nn.Parameter(torch.zeros(5000, device=dev)) for _ in range(3)]
        for k, p in enumerate(ps):
            p.grad = torch.full_like(p, 0.5 + k)
        ps[1].grad[4321] = value
        return ps
    a, b = params(), params()
    na = T.clip_grad_norm_(a, 1.0, norm_type=kind)
    nb = torch.nn.utils.clip_grad_norm_(b, 1.0, norm_type=kind)
    assert torch.equal(na.isnan(), nb.isnan()) and (bool(na.isnan()) or float(na) == float(nb))
    for p, q in zip(a, b):
        assert torch.equal(p.grad.isnan(), q.grad.isnan()) and torch.equal(p.grad.nan_to_num(), q.grad.nan_to_num())
    c = params()
    with pytest.raises(RuntimeError):
        T.clip_grad_norm_(c, 1.0, norm_type=kind, error_if_nonfinite=True)
    assert float(c[0].grad[0]) == 0.5


@gpu
def test_clip_refuses_a_tensor_named_twice(dev):
    """in place and into `out`, with and without gaps between its elements; what is only read may be named as often as one likes"""
    buf = torch.randn(64, 8, device=dev)
    for t in (buf, buf[:, ::2], buf.t()):
        before = buf.clone()
        with pytest.raises(NphmAmdError, match="share memory"):
            T.clip_grads([t, t], 0.1)
        with pytest.raises(NphmAmdError, match="share memory"):
            T.clip_grads([buf + 1, buf + 2] if t is buf else [t + 1, t + 2], 0.1, out=[t, t])
        assert torch.equal(buf, before)
        norm, (a, b) = T.clip_grads([t, t], 0.1, out=[torch.empty_like(t, memory_format=torch.contiguous_format) for _ in range(2)])
        assert abs(float(norm) - float(t.double().norm()) * 2 ** 0.5) <= float(norm) * 2.0 ** -22 and torch.equal(a, b)
    halves = buf.clone()
    T.clip_grads([halves[:, ::2], halves[:, 1::2]], 0.1)              # interleaved, but no element twice
    within(halves, buf.double() * (0.1 / (buf.double().norm() + 1e-6)), buf.double().abs() * 4 * F32)


@gpu
def test_clip_refuses_what_meets_itself_before_it_writes(dev):
    """expanded or unfolded tensors to be written: refused, with the tensors in front of them as they were; read they count as what they hold"""
    base = torch.randn(6, 8, device=dev)
    for shared in (base[:1].expand(4, 8), base[:, :1].expand(6, 5), base.view(-1).unfold(0, 8, 3), base.view(-1).as_strided((3, 4), (2, 3))):
        other, kept = torch.ones(50, device=dev), base.clone()
        with pytest.raises(NphmAmdError, match="in one place"):
            T.clip_grads([other, shared], 0.1)
        with pytest.raises(NphmAmdError, match="in one place"):
            T.clip_grads([other, torch.ones(shared.shape, device=dev)], 0.1, out=[other, shared])
        assert torch.equal(base, kept) and torch.equal(other, torch.ones(50, device=dev))
        out = torch.zeros(shared.shape, device=dev)
        norm, _ = T.clip_grads([shared], 0.1, out=[out])
        want = shared.double() * min(1.0, 0.1 / (float(shared.double().norm()) + 1e-6))
        within(out, want, clip_bound(want, torch.float32))
    for fine in (base.t(), base[::2, 1::3], base[:, 2:3], base.view(2, 3, 8)[:, 1].t()):
        want = fine.double() * min(1.0, 0.1 / (float(fine.double().norm()) + 1e-6))
        T.clip_grads([fine], 0.1)
        within(fine, want, clip_bound(want, torch.float32))


@gpu
def test_clip_refuses_views_with_gaps_that_share_memory(dev):
    """whatever their starts and orders, beside dense tensors and each other, in place and as results; interleaved views share nothing"""
    buf, kept = torch.randn(24, 40, device=dev), None
    spare = lambda like: torch.zeros(like.shape, device=dev)  # noqa: E731
    pairs = [(buf, buf[:, ::2]), (buf[:, ::2], buf), (buf[:, ::2], buf[:, 2::2]), (buf[:, 1::2], buf[:, ::3]), (buf[::2], buf[:, 5:9]), (buf.t()[3:], buf[5, 7:8]),
             (buf[1:, :-1], buf.view(-1)[900:]), (buf.view(-1)[7:-1:9], buf[20:])]
    for a, b in pairs:
        kept = buf.clone()
        for grads, out in (([a, b], [a, b]), ([spare(a), spare(b)], [a, b]), ([a, spare(b)], [spare(a), b]), ([spare(a), b], [a, spare(b)]),
                           ([spare(buf), a, b], [spare(buf), a, b])):
            with pytest.raises(NphmAmdError, match="share memory"):
                T.clip_grads(grads, 1e-3, out=out)
        with pytest.raises(NphmAmdError, match="share memory"):
            T.clip_grads([a, b], 1e-3)
        assert torch.equal(buf, kept)
        assert abs(float(T.grad_norm([a, b])) - math.hypot(float(a.double().norm()), float(b.double().norm()))) <= 4 * F32 * 2 * float(buf.norm())
    for views in ([buf[:, ::2], buf[:, 1::2]], [buf[:, :15], buf[:, 15:]], [buf[::3, ::2], buf[1::3], buf[2::3, 3:], buf[::3, 1::2]], [buf.t()[:7], buf.t()[7:].t()]):
        kept, before = buf.clone(), [v.double() for v in views]
        total = math.sqrt(sum(float(v.square().sum()) for v in before))
        norm, out = T.clip_grads(views, 0.5 * total)
        assert abs(float(norm) - total) <= 4 * F32 * total
        for v, w in zip(out, before):
            want = w * (0.5 * total / (total + 1e-6))
            within(v, want, clip_bound(want, torch.float32))
        buf.copy_(kept)
    # the two halves of one buffer
    square = torch.randn(16, 16, device=dev)
    T.clip_grads([square[:, :8]], 1e9, out=[square[:, 8:]])
    assert torch.equal(square[:, 8:], square[:, :8])


@gpu
def test_norm_of_huge_and_tiny_gradients(dev):
    """squares of these leave fp32 on both sides; the norm does not"""
    for v in (1e30, 1e-30):
        g = torch.full((10000,), v, device=dev)
        assert abs(float(T.grad_norm([g])) / float(g[0].double() * 100) - 1) <= 1e-6
        got = T.clip_grads([g.clone()], 1.0)[1][0]
        f = min(1.0, 1.0 / (100 * float(g[0].double()) + 1e-6))
        assert float((got.double() / (g.double() * f) - 1).abs().max()) <= 4 * F32
    with pytest.raises(AssertionError):          # (the plain fp32 form does)
        assert math.isfinite(float(torch.full((10000,), 1e30, device=dev).square().sum()))


@gpu
def test_clip_of_a_tensor_behind_32_bits(dev):
    """2^31 + 13 bf16 values: more than one piece of the launch's table"""
    n = (1 << 31) + 13
    g = torch.empty(n, dtype=torch.bfloat16, device=dev).normal_()
    total = math.sqrt(math.fsum(float(c.double().square().sum()) for c in g.split(1 << 27)))
    out = torch.zeros_like(g)
    norm, _ = T.clip_grads([g[:5], g[5:]], 3.0, out=[out[:5], out[5:]])
    assert abs(float(norm) - total) <= total * 1.01 * F32
    f = 3.0 / (total + 1e-6)
    for a, b in zip(g.split(1 << 27), out.split(1 << 27)):
        within(b, a.double() * f, clip_bound(a.double() * f, torch.bfloat16))


@gpu
def test_clip_sparse_and_dense_gradients_together(dev):
    """rows that an index names twice count as their sum, on both kinds of sparse tensors; the gradient stays the same tensor in dense form"""
    for coalesced in (False, True):
        gen = torch.Generator(device=dev).manual_seed(4)
        table, w = torch.nn.Parameter(torch.zeros(50, 136, device=dev)), torch.nn.Parameter(torch.zeros(70, 30, device=dev))
        idx = torch.tensor([[3, 49, 3, 0, 3, 7, 49]], device=dev)
        s = torch.sparse_coo_tensor(idx, torch.randn(7, 136, device=dev, generator=gen), (50, 136))
        table.grad = s.coalesce() if coalesced else s
        w.grad = torch.randn(70, 30, device=dev, generator=gen)
        unused = torch.nn.Parameter(torch.zeros(3, device=dev))
        dense = table.grad.to_dense().double()
        want_w = w.grad.double().clone()
        total = math.sqrt(float(dense.square().sum()) + float(want_w.square().sum()))
        # the magnitudes that a row's sum is made of: of the entries as they come in (the call works on them in place; read after it
        # they are f times smaller, and the bound f^2 mag where f mag is meant)
        mag = torch.zeros(50, 136, dtype=torch.float64, device=dev).index_add_(0, idx[0], s._values().abs().double())
        norm = T.clip_grad_norm_(iter([table, unused, w]), 2.0)
        assert abs(float(norm) - total) <= total * 8 * F32            # (a row's sum is rounded before its square)
        f = 2.0 / (total + 1e-6)
        within(table.grad.to_dense(), dense * f, mag * f * 8 * F32 + 1e-30)
        within(w.grad, want_w * f, want_w.abs() * f * 12 * F32)


@gpu
@pytest.mark.parametrize("N,rows,D", [(200, 7, 33), (700, 50, 8), (9000, 300, 20), (30000, 3, 5), (20000, 100000, 4)])
def test_duplicates_of_a_sparse_gradient_are_folded(dev, N, rows, D):
    """every entry's row in order: the first entry of a row holds the sum of its entries (fp32, in their order), the others zeros"""
    gen = torch.Generator(device=dev).manual_seed(N)
    idx = (torch.rand(N, device=dev, generator=gen) ** 2 * rows).long().clamp_(0, rows - 1)
    values = torch.randn(N, D, device=dev, generator=gen)
    s = torch.sparse_coo_tensor(idx[None], values.clone(), (rows, D))
    T._merge_rows_(s)
    got = s._values()
    want = torch.zeros(rows, D, dtype=torch.float64, device=dev).index_put_((idx,), values.double(), accumulate=True)
    mag = torch.zeros(rows, D, dtype=torch.float64, device=dev).index_put_((idx,), values.double().abs(), accumulate=True)
    many = torch.bincount(idx, minlength=rows)[:, None].double()
    first = torch.full((rows,), N, device=dev).scatter_reduce_(0, idx, torch.arange(N, device=dev), "amin")
    heads = first[many[:, 0] > 0]
    within(got[heads], want[idx[heads]], (mag * (many + 1) * F32)[idx[heads]] + 1e-30)
    rest = torch.ones(N, dtype=torch.bool, device=dev)
    rest[heads] = False
    assert not got[rest].any()


@gpu
@pytest.mark.parametrize("asks", [False, True])
def test_forward_mode_inputs_are_refused(dev, asks):
    """a dual tensor would come out without its tangent; whether it requires a gradient or not, in every place that takes one"""
    import torch.autograd.forward_ad as fwAD
    idx = torch.tensor([1, 0], device=dev)
    plain = lambda *s, t=torch.bfloat16: torch.randn(*s, device=dev).to(t)  # noqa: E731
    with fwAD.dual_level():
        dual = lambda *s, t=torch.bfloat16: fwAD.make_dual(plain(*s, t=t).requires_grad_(asks), plain(*s, t=t))  # noqa: E731
        table, x, w, b, r = dual(4, 8, t=torch.float32), dual(3, 8), dual(5, 8), dual(5), dual(3, 5)
        for call in (lambda: T.lookup_rows(table, idx), lambda: T.lookup_rows(table, idx, sparse=True), lambda: T.lookup_rows_grad(table[:2], idx, 4),
                     lambda: T.renorm_rows_(table, idx, 1e-3), lambda: T.linear_act(x, plain(5, 8)), lambda: T.linear_act(plain(3, 8), w, activation="relu"),
                     lambda: T.linear_act(plain(3, 8), plain(5, 8), b), lambda: T.linear_act(plain(3, 8), plain(5, 8), residual=r),
                     lambda: T.grad_norm([plain(3), w]), lambda: T.clip_grads([w], 1.0, out=[plain(5, 8)]), lambda: T.clip_grads([plain(5, 8)], 1.0, out=[w])):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            T.linear_act(x, plain(5, 8))
        leaf, codes = plain(5, 8).requires_grad_(), plain(4, 8).requires_grad_()
        for y, p in ((T.linear_act(plain(3, 8), leaf), leaf), (T.lookup_rows(codes, idx), codes), (T.lookup_rows(codes, idx, sparse=True), codes)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(y, p, fwAD.make_dual(plain(*y.shape), plain(*y.shape)))
    T.lookup_rows(plain(4, 8), idx)


def dirty_memory(dev):
    """small blocks that are handed out again hold NaN: what a later call leaves unwritten shows"""
    held = [torch.full((n * 1344,), math.nan, device=dev) for n in (1, 2, 3, 4, 6, 8, 12, 24) for _ in range(4)]
    torch.cuda.synchronize()
    del held


def sparse_adam_bound(steps, lr, w):
    """A step of Adam adds lr sqrt(1 - b2^t) / (1 - b1^t) m / (sqrt(v) + eps) to an entry: 0.316 lr m / sqrt(v) at most, the factor's largest
    value that of t = 1.  m comes from eight fp32 roundings of magnitudes up to the largest gradient's, sqrt(v) is at least 0.0316 of that
    (its last one's share), so the two sides are 2 x 8 x 2^-24 x 0.316 / 0.0316 lr apart, and a rounding of the sum."""
    return steps * (160 * lr * F32 + float(w.abs().max()) * F32)


@gpu
@pytest.mark.parametrize("D", [200, 256, 257, 300, 513, 1344, 2048])
@pytest.mark.parametrize("way", ["plain", "clipped", "twice", "summed", "embedding", "copied"])
def test_row_gradients_step_sparse_adam(dev, way, D):
    """three steps of the trainer's optimiser on codes of this width, against the same optimiser on the host, which is handed the gradient in its
    dense form: no column is lost, whether the gradient is one call's, clipped, of two calls, summed over two backward passes, or torch's"""
    import copy
    gen = torch.Generator().manual_seed(D)
    start = torch.randn(9, D, generator=gen) * 0.01
    codes = (torch.nn.Embedding(9, D, sparse=True) if way == "embedding" else T.LatentCodes(9, D, sparse=True)).to(dev)
    with torch.no_grad():
        codes.weight.copy_(start)
    if way == "copied":
        codes = copy.deepcopy(codes)
    host = torch.nn.Parameter(start.clone())
    ours, ref = torch.optim.SparseAdam([codes.weight], lr=1e-3), torch.optim.SparseAdam([host], lr=1e-3)
    for k, idx in enumerate(([3, 1, 3, 0], [5, 0, 5], [1, 3, 8, 7, 3])):
        idx = torch.tensor(idx)
        go = torch.randn(len(idx), D, generator=gen)
        mags = torch.zeros(9, D).index_add_(0, idx, go.abs())
        want = torch.zeros(9, D, dtype=torch.float64).index_add_(0, idx, go.double())
        dirty_memory(dev)
        codes.weight.grad = None
        if way == "twice":
            ((codes(idx.to(dev)) * go.to(dev)).sum() * 0.25 + (codes(idx.to(dev)) * go.to(dev)).sum() * 0.75).backward()
        elif way == "summed":
            for f in (0.25, 0.75):
                ((codes(idx.to(dev)) * go.to(dev)).sum() * f).backward()
        else:
            (codes(idx.to(dev)) * go.to(dev)).sum().backward()
        if way in ("clipped", "embedding"):
            norm = float(T.clip_grad_norm_(codes.parameters(), 0.5))
            assert abs(norm - float(want.norm())) <= 16 * F32 * float(mags.double().norm())
            want, mags = want * (0.5 / (norm + 1e-6)), mags * (0.5 / (norm + 1e-6))
        g = codes.weight.grad
        assert g.is_sparse and (D <= 256 or g.is_coalesced())
        dense = g.to_dense().cpu()
        within(dense, want, mags.double() * 24 * F32 + 1e-30)            # (two products, four sums and the factor's six roundings, each on either way)
        rows = torch.unique(idx)
        host.grad = torch.sparse_coo_tensor(rows[None], dense[rows], (9, D))
        dirty_memory(dev)
        ours.step()
        ref.step()
        assert float((codes.weight.detach().cpu() - host.detach()).abs().max()) <= sparse_adam_bound(k + 1, 1e-3, start), k


@gpu
@pytest.mark.parametrize("D", [40, 300])
@pytest.mark.parametrize("kind", [torch.int64, torch.int32])
def test_padding_in_a_batch_moves_no_row_of_a_sparse_table(dev, D, kind):
    """row 0 has momentum from the first step; the batches behind it name padding and other rows, or padding alone: it keeps its bits, and so
    does the padding row"""
    codes = T.LatentCodes(6, D, padding_idx=-2, sparse=True, device=dev)
    assert codes.padding_idx == 4
    optim = torch.optim.SparseAdam(codes.parameters(), lr=1e-2)
    kept = None
    for idx in ([0, 4, 1, 0], [4, 2, 4], [4, 4], [4], [5, 4]):
        optim.zero_grad()
        before = codes.weight.detach().clone()
        codes(torch.tensor(idx, device=dev, dtype=kind)).square().sum().add(codes.weight[0, 0].detach()).backward()
        optim.step()
        named = sorted(set(idx) - {4})
        moved = [v for v in range(6) if not torch.equal(codes.weight[v], before[v])]
        if kept is None:
            kept = codes.weight[0].detach().clone()
        assert torch.equal(codes.weight[0], kept) and set(moved) <= set(named), (idx, moved)
        assert bool(torch.isfinite(codes.weight).all())


@gpu
@pytest.mark.parametrize("sparse", [False, True])
def test_pretrained_codes_look_up_and_learn(dev, sparse):
    rows = torch.randn(7, 300, device=dev)
    idx = torch.tensor([[2, 2], [6, 0]], device=dev)
    codes, ref = T.LatentCodes.from_pretrained(rows.clone(), freeze=False, sparse=sparse), torch.nn.Embedding.from_pretrained(rows.clone(), freeze=False)
    go = torch.randn(2, 2, 300, device=dev)
    a, b = codes(idx), ref(idx)
    assert torch.equal(a, b)
    a.backward(go)
    b.backward(go)
    assert codes.weight.grad.is_sparse == sparse
    got = codes.weight.grad.to_dense() if sparse else codes.weight.grad
    mags = torch.zeros_like(got).index_add_(0, idx.view(-1), go.view(-1, 300).abs()).double()
    within(got, ref.weight.grad.double(), 4 * F32 * mags)
    assert not T.LatentCodes.from_pretrained(rows)(idx).requires_grad


@gpu
@pytest.mark.parametrize("t", FLOATS)
def test_a_folded_row_gradient_holds_every_row_once(dev, t):
    gen = torch.Generator(device=dev).manual_seed(2)
    for V, shape, N in ((1, (300,), 5), (70, (257,), 1), (70, (3, 200), 900), (50000, (300,), 9001)):
        idx = (torch.rand(N, device=dev, generator=gen) ** 2 * V).long().clamp_(0, V - 1)
        values = torch.randn(N, *shape, device=dev, generator=gen).to(t)
        g = torch.sparse_coo_tensor(idx[None], values, (V, *shape), is_coalesced=False)
        assert T._needs_fold(g)
        f = T._folded(g)
        assert f.is_coalesced() and f.dtype == t and f.shape == g.shape and not T._needs_fold(f)
        rows = torch.unique(idx.cpu())
        assert torch.equal(f._indices()[0].cpu(), rows)
        want = torch.zeros(V, *shape, dtype=torch.float64, device=dev).index_put_((idx,), values.double(), accumulate=True)[rows.to(dev)]
        mag = torch.zeros(V, *shape, dtype=torch.float64, device=dev).index_put_((idx,), values.double().abs(), accumulate=True)[rows.to(dev)]
        within(f._values(), want, want.abs() * half_step(t) * (1 + half_step(t)) + mag * N * F32 + tiny(t))
    assert not T._needs_fold(torch.sparse_coo_tensor(idx[None], values[:, :256], (V, 256)))      # torch takes these itself


@gpu
def test_every_stage_of_the_training_script_stays_finite(dev):
    """the trainer's step; after each stage the code table, its gradient and the optimiser's state hold finite numbers, and what a stage does not
    write keeps its bits"""
    from nphm_amd.loss_functions import compute_loss, weighted_total
    decoder = U.build_identity(device=dev).train()
    gen = torch.Generator().manual_seed(13)
    B = 4
    pts = lambda n: (torch.rand(B, n, 3, generator=gen) - 0.5) * 0.5  # noqa: E731
    nrm = lambda n: torch.nn.functional.normalize(torch.randn(B, n, 3, generator=gen), dim=-1)  # noqa: E731
    batch = {"points_face": pts(60), "normals_face": nrm(60), "points_non_face": pts(9), "normals_non_face": nrm(9), "sup_grad_far": nrm(11) * 0.4,
             "sup_grad_near": pts(33), "gt_anchors": torch.from_numpy(U.anchors_mean()).float().reshape(1, 39, 3).repeat(B, 1, 1),
             "idx": torch.tensor([[3], [1], [3], [0]]), "path": ["x"] * B}
    lambdas = {"surf_sdf": 2.0, "normals": 0.3, "space_sdf": 0.01, "grad": 0.1, "lat_reg": 0.005, "anchors": 7.5, "symm_dist": 0.005, "middle_dist": 0.001}
    codes = T.LatentCodes(6, decoder.lat_dim, max_norm=1.0, sparse=True, device=dev)
    with torch.no_grad():
        codes.weight.copy_(torch.randn(6, decoder.lat_dim, generator=gen) * 0.1)
    optims = torch.optim.AdamW(decoder.parameters(), lr=1e-4), torch.optim.SparseAdam(codes.parameters(), lr=1e-3)
    idle = codes.weight.detach()[[2, 4, 5]].clone()

    def finite(stage, *tensors):
        for t in tensors:
            assert bool(torch.isfinite(t).all()), (stage, (~torch.isfinite(t)).nonzero()[:4].tolist())

    for k in range(3):
        dirty_memory(dev)
        for o in optims:
            o.zero_grad()
        loss = weighted_total(compute_loss(dict(batch), decoder, codes, dev), lambdas)
        finite("forward", loss.detach(), codes.weight.detach())
        dirty_memory(dev)
        loss.backward()
        finite("backward", codes.weight.grad._values(), *[p.grad for p in decoder.parameters() if p.grad is not None])
        norms = T.clip_grad_norm_(decoder.parameters(), 0.1), T.clip_grad_norm_(codes.parameters(), 0.1)
        grad = codes.weight.grad
        finite("clips", *norms, grad._values(), *[p.grad for p in decoder.parameters() if p.grad is not None])
        assert grad._indices()[0].tolist() == [0, 1, 3]
        table, values = codes.weight.detach().clone(), grad._values().clone()
        dirty_memory(dev)
        optims[0].step()
        assert torch.equal(codes.weight, table) and torch.equal(grad._values(), values)
        optims[1].step()
        state = optims[1].state[codes.weight]
        finite("optimisers", codes.weight.detach(), state["exp_avg"], state["exp_avg_sq"])
        assert float((codes.weight.detach() - table).abs().max()) <= 3.2e-3           # (Adam's largest step: lr (1 - b1) / sqrt(1 - b2))
        assert torch.equal(codes.weight.detach()[[2, 4, 5]], idle)
        assert not bool(state["exp_avg"][[2, 4, 5]].any()) and not bool(state["exp_avg_sq"][[2, 4, 5]].any())


# ---- all of them -----------------------------------------------------------------------------------------------------------------

def step(dev, codes, layers, idx, pts, target):
    """codes -> two residual layers -> loss -> gradients, clipped by one norm"""
    x = torch.cat([codes(idx), pts], -1).to(torch.bfloat16)
    h = T.linear_act(x, layers[0], layers[1], "softplus", 10.0)
    h = T.linear_act(h, layers[2], layers[3], "silu", residual=h)
    loss = (h.float() - target).square().mean()
    for p in (codes.weight, *layers):
        p.grad = None
    loss.backward()
    return loss, T.clip_grad_norm_([codes.weight, *layers], 0.05)


def step_inputs(dev, sparse):
    gen = torch.Generator(device=dev).manual_seed(11)
    codes = T.LatentCodes(20, 61, max_norm=1.0, sparse=sparse, device=dev)
    with torch.no_grad():
        codes.weight.copy_(torch.randn(20, 61, device=dev, generator=gen) * 0.2)
    layers = [(torch.randn(*s, device=dev, generator=gen) * 0.15).bfloat16().requires_grad_() for s in ((128, 64), (128,), (128, 128), (128,))]
    idx = torch.randint(0, 20, (96,), device=dev, generator=gen)
    return codes, layers, idx, torch.randn(96, 3, device=dev, generator=gen), torch.randn(96, 128, device=dev, generator=gen)


@gpu
@pytest.mark.parametrize("sparse", [False, True])
def test_a_step_of_all_operators(dev, sparse):
    """against the same step in fp64.  bf16 roundings on the way of a gradient entry: x, z, y, z, y, g, gz, dh, gz, dx - ten of 2^-8 / 2 each if
    they all add up in one direction; as they do not, the 2-norm of each gradient is held to ten half steps of its 2-norm, and
    clipping to the norm found"""
    codes, layers, idx, pts, target = step_inputs(dev, sparse)
    start = codes.weight.detach().double()
    loss, norm = step(dev, codes, layers, idx, pts, target)
    named = torch.unique(idx)
    n = start[named].norm(dim=1, keepdim=True)
    start[named] = torch.where(n > 1, start[named] / (n + 1e-7), start[named])
    assert float((codes.weight.detach().double() - start).abs().max()) <= 4 * F32
    t, ls = start.clone().requires_grad_(), [p.detach().double().requires_grad_() for p in layers]
    x = torch.cat([t[idx], pts.double()], -1)
    h = torch.nn.functional.softplus(x @ ls[0].t() + ls[1], beta=10.0)
    h = torch.nn.functional.silu(h @ ls[2].t() + ls[3]) + h
    ref = (h - target.double()).square().mean()
    grads = torch.autograd.grad(ref, [t, *ls])
    total = math.sqrt(sum(float(g.square().sum()) for g in grads))
    room = 10 * 2.0 ** -9
    assert abs(float(loss) - float(ref)) <= room * float(ref)
    assert abs(float(norm) - total) <= room * total
    for p, g in zip([codes.weight, *layers], grads):
        own = (p.grad.to_dense() if p.grad.is_sparse else p.grad).double()
        f = 0.05 / (total + 1e-6)
        assert float((own - g * f).norm()) <= 2 * room * float((g * f).norm())
    assert abs(float(T.grad_norm([p.grad.coalesce().values() if p.grad.is_sparse else p.grad for p in (codes.weight, *layers)])) - 0.05) <= 0.05 * 2.0 ** -9


@gpu
def test_training_script_with_the_operators(dev):
    """training.py's step (compute_loss, backward, two clips, AdamW + SparseAdam) with LatentCodes and clip_grad_norm_ in place of nn.Embedding and
    torch's clip, which takes no sparse gradient: losses of the same first step, and a code gradient of the same norm"""
    from nphm_amd.loss_functions import compute_loss
    decoder = U.build_identity(device=dev).train()
    gen = torch.Generator().manual_seed(11)
    B, box = 4, torch.tensor([0.5, 0.6, 0.5])
    pts = lambda n: (torch.rand(B, n, 3, generator=gen) - 0.5) * box + torch.tensor([0.0, 0.05, 0.05])  # noqa: E731
    nrm = lambda n: torch.nn.functional.normalize(torch.randn(B, n, 3, generator=gen), dim=-1)  # noqa: E731
    face, non = pts(96), pts(8)
    batch = {"points_face": face, "normals_face": nrm(96), "points_non_face": non, "normals_non_face": nrm(8), "sup_grad_far": nrm(12) * 0.4,
             "sup_grad_near": torch.cat([face, non], 1) + 0.01 * torch.randn(B, 104, 3, generator=gen),
             "gt_anchors": torch.from_numpy(U.anchors_mean()).float().reshape(1, 39, 3).repeat(B, 1, 1),
             "idx": torch.tensor([[3], [1], [3], [0]]), "path": ["x"] * B}
    lambdas = {"surf_sdf": 2.0, "normals": 0.3, "space_sdf": 0.01, "grad": 0.1, "lat_reg": 0.005, "anchors": 7.5, "symm_dist": 0.005, "middle_dist": 0.001}
    start = torch.randn(6, decoder.lat_dim, generator=gen).to(dev) * 0.1
    seen = []
    for kind in (T.LatentCodes, torch.nn.Embedding):
        codes = kind(6, decoder.lat_dim, max_norm=1.0, sparse=True).to(dev)
        with torch.no_grad():
            codes.weight.copy_(start)
        decoder.zero_grad()
        losses = compute_loss(dict(batch), decoder, codes, dev)
        sum(lambdas[k] * losses[k] for k in losses).backward()
        norm = T.clip_grad_norm_(codes.parameters(), 1e-4)
        dense = codes.weight.grad.to_dense()
        assert abs(float(dense.double().norm()) - 1e-4) <= 1e-4 * 0.02           # (1e-6 beside a norm of 1e-4 in the factor's formula)
        seen.append(({k: float(v.detach()) for k, v in losses.items()}, float(norm), codes))
    for k, v in seen[1][0].items():
        assert abs(seen[0][0][k] - v) <= 2e-5 * max(1.0, abs(v)), k
    assert abs(seen[0][1] - seen[1][1]) <= 1e-3 * seen[1][1]
    norm = T.clip_grad_norm_(decoder.parameters(), 0.1)
    assert math.isfinite(float(norm))
    torch.optim.AdamW(decoder.parameters(), lr=1e-4).step()
    torch.optim.SparseAdam(list(seen[0][2].parameters()), lr=1e-3).step()
    assert bool(torch.isfinite(seen[0][2].weight).all())


@gpu
def test_a_captured_step_replays_as_the_eager_one(dev):
    """graph and eager steps in turn, new inputs each time: the same bits (the graph has its own leaves: none is shared with an eager graph)"""
    codes, layers, idx, pts, target = step_inputs(dev, False)
    own = T.LatentCodes(20, 61, max_norm=1.0, device=dev)
    own.load_state_dict(codes.state_dict())
    own_layers = [p.detach().clone().requires_grad_() for p in layers]
    s_idx, s_pts = idx.clone(), pts.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(dev, own, own_layers, s_idx, s_pts, target)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    for p in (own.weight, *own_layers):
        p.grad = None
    with torch.cuda.graph(graph):
        _, norm = step(dev, own, own_layers, s_idx, s_pts, target)
    for k in range(4):
        s_idx.copy_((idx + k) % 20)
        s_pts.copy_(pts * (1 + k))
        graph.replay()
        torch.cuda.synchronize()
        _, want = step(dev, codes, layers, s_idx.clone(), s_pts.clone(), target)
        torch.cuda.synchronize()
        assert torch.equal(norm, want)
        for p, q in zip((own.weight, *own_layers), (codes.weight, *layers)):
            assert torch.equal(p.grad, q.grad) and torch.equal(p, q)


@gpu
@pytest.mark.parametrize("op", ["layer", "lookup", "sparse lookup"])
def test_a_captured_pass_into_an_eager_graphs_leaf_is_refused(dev, op):
    """raised before autograd would add the gradient on the default stream; once the eager graph is gone the same capture goes through"""
    idx, g = torch.tensor([1, 0, 1], device=dev), torch.randn(3, 8, device=dev)
    leaf = (torch.randn(8, 8, device=dev).bfloat16() if op == "layer" else torch.randn(4, 8, device=dev)).requires_grad_()
    x = torch.randn(3, 8, device=dev).bfloat16()
    call = {"layer": lambda: T.linear_act(x, leaf, activation="silu"), "lookup": lambda: T.lookup_rows(leaf, idx),
            "sparse lookup": lambda: T.lookup_rows(leaf, idx, sparse=True)}[op]
    g = g.to(leaf.dtype)
    alive = call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(NphmAmdError, match="eager calls"):
            try:
                call().backward(g)
            except RuntimeError as e:                                # (autograd raises it: known by its text)
                raise NphmAmdError(str(e)) from None
    assert leaf.grad is None
    alive.backward(g)
    want = leaf.grad.to_dense() if leaf.grad.is_sparse else leaf.grad
    leaf.grad = None
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call().backward(g)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(leaf.grad.to_dense() if leaf.grad.is_sparse else leaf.grad, want)
        leaf.grad._values().zero_() if leaf.grad.is_sparse else leaf.grad.zero_()        # (written again by the next replay)


@gpu
def test_a_captured_step_of_a_wide_sparse_table(dev):
    """inside a graph the gradient keeps an entry for every index (nothing can wait there), its duplicates folded by the clip: the same gradient as
    the eager step's coalesced one, which the clip outside makes of it"""
    gen = torch.Generator(device=dev).manual_seed(5)
    start = torch.randn(12, 300, device=dev, generator=gen) * 0.1
    own, eager = [T.LatentCodes(12, 300, max_norm=1.0, sparse=True, device=dev) for _ in range(2)]
    idx, go = torch.tensor([3, 1, 3, 0, 3], device=dev), torch.randn(5, 300, device=dev, generator=gen)
    s_idx, s_go = idx.clone(), go.clone()

    def run(codes, i, g):
        codes.weight.grad = None
        codes(i).backward(g)
        return T.clip_grad_norm_(codes.parameters(), 0.7)

    for codes in (own, eager):
        with torch.no_grad():
            codes.weight.copy_(start)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(own, s_idx, s_go)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = run(own, s_idx, s_go)
    captured = own.weight.grad
    for k in range(4):
        s_idx.copy_((idx + k) % 12)
        s_go.copy_(go * (1 + k))
        graph.replay()
        torch.cuda.synchronize()
        want = run(eager, s_idx.clone(), s_go.clone())
        torch.cuda.synchronize()
        mag = torch.zeros(12, 300, dtype=torch.float64, device=dev).index_add_(0, s_idx, s_go.abs().double()) * (0.7 / float(want))
        assert abs(float(norm) - float(want)) <= 8 * F32 * float(want)
        assert eager.weight.grad.is_coalesced() and not captured.is_coalesced() and captured._nnz() == 5
        within(captured.to_dense(), eager.weight.grad.to_dense().double(), mag * 16 * F32 + 1e-30)
        assert torch.equal(own.weight, eager.weight)
    before = captured.to_dense()
    own.weight.grad = captured
    T.clip_grad_norm_(own.parameters(), 1e9)
    assert own.weight.grad.is_coalesced() and float((own.weight.grad.to_dense() - before).abs().max()) <= 2 * F32 * float(before.abs().max())


@gpu
def test_operators_run_on_the_current_stream(dev):
    """work queued behind a long product on another stream: the operators wait for it there, and two streams at once do not meet"""
    x, w, b, r, g = layer_inputs(dev, torch.bfloat16, 256, 256, 256, True, True)
    table = torch.randn(500, 256, device=dev)
    idx = torch.randint(0, 500, (3000,), device=dev)
    rows = torch.randn(3000, 256, device=dev)
    want = T.linear_act(x, w, b, "silu", residual=r), T.lookup_rows_grad(rows, idx, 500), T.clip_grads([rows], 1.0, out=[torch.empty_like(rows)])[1][0]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            big = torch.randn(4096, 4096, device=dev)
            big = big @ big
            late = torch.zeros_like(x).copy_(x)
            late_rows = torch.zeros_like(rows).copy_(rows)
            got.append((T.linear_act(late, w, b, "silu", residual=r), T.lookup_rows_grad(late_rows, idx, 500),
                        T.clip_grads([late_rows], 1.0, out=[torch.empty_like(rows)])[1][0]))
    torch.cuda.synchronize()
    for trio in got:
        assert all(torch.equal(a, b_) for a, b_ in zip(trio, want))
