"""The token-side operators (embedding, LayerNorm, token log probabilities) against
their definitions in 64 bits.

Tolerances are elementwise bounds computed from the data: u = 2^-24 is half a
step of fp32, a sum of k terms in a chain errs by at most k u of the terms'
absolute sum, an output in a narrower type adds half a step of it
(``torch.finfo(t).eps / 2``).  Where the data are small integers every sum is
exact in any order, and the comparison is equality.
"""

import ctypes

import pytest
import torch

from spikingtransformer_b200 import _lib

DEV = "cuda"
U = 2.0 ** -24
FLOATS = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    from spikingtransformer_b200 import ops as o
    return o


def gen(seed):
    return torch.Generator().manual_seed(seed)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the spacing of the type's subnormal numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def assert_within(got, want, bound, what):
    got, want, bound = got.detach().double().cpu(), want.detach().double().cpu(), bound.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - bound
    worst = over.max().item() if over.numel() else -1.0
    assert worst <= 0, "%s: %.3e over its bound (error %.3e)" % (what, worst, (got - want).abs().max().item())


# ------------------------------------------------------------------ refusals without a device


def test_c_entries_reject_bad_arguments():
    lib = _lib.load()
    p = ctypes.c_void_p(16)  # never dereferenced: the checks come first
    assert lib.spk_layer_norm_fwd(None, 0, 8, None, 0, None, 0, 1e-5, 2, 8, p, 0, None, None) == 1
    assert lib.spk_layer_norm_fwd(p, 3, 8, None, 0, None, 0, 1e-5, 2, 8, p, 0, None, None) == 1   # u8
    assert lib.spk_layer_norm_fwd(p, 0, 7, None, 0, None, 0, 1e-5, 2, 8, p, 0, None, None) == 2   # ld < D
    assert lib.spk_layer_norm_fwd(p, 0, 8, None, 0, None, 0, 1e-5, 0, 8, p, 0, None, None) == 2   # no rows
    assert lib.spk_layer_norm_bwd(p, 0, p, 0, 8, None, p, 0, 2, 8, p, p, p, 0, p, 1 << 30, None) == 1
    assert lib.spk_layer_norm_bwd(p, 0, p, 0, 8, p, p, 0, 2, 8, p, p, p, 0, p, 4, None) == 1      # workspace
    tail = (-1, None, 0, None)
    assert lib.spk_embedding_fwd(p, p, 0, 8, 1.0, 4, 10, 8, p, 0, None, *tail) == 1
    assert lib.spk_embedding_fwd(p, p, 0, 7, 1.0, 4, 10, 8, p, 0, p, *tail) == 2
    assert lib.spk_embedding_fwd(p, p, 5, 8, 1.0, 4, 10, 8, p, 0, p, *tail) == 1
    assert lib.spk_embedding_fwd(p, p, 0, 8, 1.0, 4, 10, 8, p, 0, p, -1, p, 63, None) == 1        # plan: 4 tokens
    assert lib.spk_embedding_bwd(p, p, 0, 1.0, -1, 4, 0, 8, p, 0, p, 1 << 30, p, 1 << 30, None) == 2
    assert lib.spk_embedding_bwd(p, p, 0, 1.0, -1, 4, 10, 8, p, 0, p, 63, p, 1 << 30, None) == 1  # plan
    assert lib.spk_embedding_bwd(p, p, 0, 1.0, -1, 4, 10, 8, p, 0, p, 64, p, 0, None) == 1        # workspace
    assert lib.spk_embedding_bwd(p, p, 0, 1.0, -1, 4, 10, 8, p, 0, None, 64, p, 1 << 30, None) == 1
    args = (p, p, p, p, p, p, p, 1 << 30, None)
    assert lib.spk_token_logprobs_fwd(None, 0, 1, 2, 8, 0, 8, p, -100, 0, *args) == 1
    assert lib.spk_token_logprobs_fwd(p, 3, 1, 2, 8, 0, 8, p, -100, 0, *args) == 1
    assert lib.spk_token_logprobs_fwd(p, 0, 1, 2, 8, 0, 8, p, -100, 9, *args) == 2                # top_k > V
    assert lib.spk_token_logprobs_fwd(p, 0, 1, 2, 99, 0, 99, p, -100, 33, *args) == 2             # top_k > 32
    assert lib.spk_token_logprobs_fwd(p, 0, 1, 2, 99999, 0, 99999, p, -100, 0, *args[:-3], p, 16, None) == 1  # workspace
    assert lib.spk_token_logprobs_fwd(p, 0, 65, 2, 8, 0, 8, p, -100, 0, *args) == 2
    assert lib.spk_token_logprobs_fwd(p, 0, 1, 2, 8, 0, -8, p, -100, 0, *args) == 2
    assert lib.spk_token_logprobs_bwd(p, 0, 1, 2, 8, 0, 8, p, -100, 4, None, p, p, p, p, p, None) == 1  # no indices


def test_ops_refuse_cpu_tensors(ops):
    x, t = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: ops.layer_norm(x), lambda: ops.embedding(t, x), lambda: ops.token_logprobs(x[None], t)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_autograd_nodes_load_and_report_their_errors(ops):
    """The compiled nodes load without a device, and refuse what has no data."""
    nodes = ops._embedding_nodes()
    assert nodes is ops._embedding_nodes()
    with pytest.raises(RuntimeError, match="data"):
        nodes.embedding(torch.empty(4, 8, device="meta"), torch.zeros(2, dtype=torch.int64, device="meta"), 1.0, -1,
                        torch.float32, 0)


@pytest.mark.gpu
def test_ops_refuse_what_they_do_not_take(ops):
    x = torch.randn(4, 8, device=DEV)
    t = torch.zeros(4, dtype=torch.int64, device=DEV)
    for call, err in [
            (lambda: ops.layer_norm(x.double()), TypeError),
            (lambda: ops.layer_norm(x, torch.ones(7, device=DEV)), RuntimeError),
            (lambda: ops.layer_norm(x, torch.ones(8)), RuntimeError),
            (lambda: ops.layer_norm(x, out_dtype=torch.uint8), TypeError),
            (lambda: ops.layer_norm(x[:, :0]), RuntimeError),
            (lambda: ops.layer_norm_bwd(x[:2], x, torch.zeros(4, 2, device=DEV)), RuntimeError),
            (lambda: ops.layer_norm_bwd(x, x, torch.zeros(3, 2, device=DEV)), RuntimeError),
            (lambda: ops.embedding(t.float(), x), TypeError),
            (lambda: ops.embedding(t, x[0]), RuntimeError),
            (lambda: ops.embedding(t, x, padding_idx=4), ValueError),
            (lambda: ops.embedding(t, x, padding_idx=-1), ValueError),
            (lambda: ops.embedding_bwd(x[:3], t, 8), RuntimeError),
            (lambda: ops.token_logprobs(x, t), RuntimeError),
            (lambda: ops.token_logprobs(x[None], t[:3]), RuntimeError),
            (lambda: ops.token_logprobs(x[None], t, top_k=9), ValueError),
            (lambda: ops.token_logprobs(x[None], t, top_k=-1), ValueError),
            (lambda: ops.token_logprobs(x[None].double(), t), TypeError),
            (lambda: ops.token_logprobs(x[None], t.bool()), TypeError)]:
        with pytest.raises(err):
            call()


@pytest.mark.gpu
def test_second_derivatives_are_refused(ops):
    x = torch.randn(4, 8, device=DEV, requires_grad=True)
    t = torch.zeros(4, dtype=torch.int64, device=DEV)
    for y in (ops.layer_norm(x), ops.token_logprobs(x[None], t)[0]):
        (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


@pytest.mark.gpu
def test_forward_mode_tangents_are_refused_and_not_lost(ops):
    """A tangent on an input, with or without a gradient wanted, or on a gradient: an
    error, as from every operator without a forward-mode derivative.  The embedding's
    gradient is linear in g and takes g's tangent through."""
    import torch.autograd.forward_ad as fwd
    x, v = torch.randn(4, 8, device=DEV), torch.randn(4, 8, device=DEV)
    w = torch.ones(8, device=DEV)
    t = torch.tensor([0, 3, 1, 3], device=DEV)
    calls = [lambda p: ops.layer_norm(p), lambda p: ops.layer_norm(x, p[0]), lambda p: ops.layer_norm(x, None, p[0]),
             lambda p: ops.embedding(t, p), lambda p: ops.token_logprobs(p[None], t)]
    with fwd.dual_level():
        for call in calls:
            for leaf in (x, x.clone().requires_grad_(True)):
                with pytest.raises(NotImplementedError):
                    call(fwd.make_dual(leaf, v))
                with pytest.raises(NotImplementedError), torch.no_grad():
                    call(fwd.make_dual(leaf, v))
            call(x)  # no tangent: as ever
        for call in (lambda p: ops.layer_norm(p), lambda p: ops.layer_norm(x, p[0]),
                     lambda p: ops.token_logprobs(p[None], t)[0]):
            leaf = x.clone().requires_grad_(True)
            y = call(leaf)
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(y, leaf, fwd.make_dual(torch.ones_like(y), torch.ones_like(y)))
        leaf = x.clone().requires_grad_(True)
        g = torch.randint(-9, 10, (4, 8), device=DEV).float()
        (gw,) = torch.autograd.grad(ops.embedding(t, leaf, 2.0)[0], leaf, fwd.make_dual(g, g + 1))
        for got, of in zip(fwd.unpack_dual(gw), (g, g + 1)):
            assert torch.equal(got.cpu().double(), scatter_exact(t.cpu(), of.cpu(), 4, 2.0))


# ------------------------------------------------------------------ LayerNorm


def ln_case(rows, D, dtype, seed, offset=1.0, w_dtype=torch.float32):
    g = gen(seed)
    x = (torch.randn(rows, D, generator=g) * 1.5 + offset * torch.randn(rows, 1, generator=g)).to(dtype)
    w = (1 + 0.3 * torch.randn(D, generator=g)).to(w_dtype)
    b = (0.3 * torch.randn(D, generator=g)).to(w_dtype)
    gy = torch.randn(rows, D, generator=g).to(dtype)
    return x, w, b, gy


def ln_exact(x, w, b, gy, eps, out_dtype):
    """The formulas and the error bounds of y, gx, gw, gb in 64 bits."""
    D = x.shape[-1]
    k = D / 32 + 16  # a thread's chain over its part of the row, and the joins
    X, G = x.double(), gy.double()
    W = torch.ones(D, dtype=torch.float64) if w is None else w.double()
    Bv = torch.zeros(D, dtype=torch.float64) if b is None else b.double()
    mean = X.mean(-1, keepdim=True)
    var = ((X - mean) ** 2).mean(-1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    h = (X - mean) * r
    y = h * W + Bv
    e_mean = (k + 1) * U * X.abs().mean(-1, keepdim=True)
    e_c = e_mean + U * (X - mean).abs()                  # of x - mean
    e_var = (2 * (X - mean).abs() * e_c + e_c ** 2).mean(-1, keepdim=True) + (k + 2) * U * var
    e_r = r * (e_var / (2 * (var + eps)) * 1.01 + 4 * U)
    e_h = r * e_c + (X - mean).abs() * e_r + 2 * U * h.abs()
    step = half_step(out_dtype)
    e_y = (e_h * W.abs() + 2 * U * (h * W).abs() + U * y.abs()) * (1 + step) + step * y.abs() + tiny(out_dtype)
    a = G * W
    ma, mh = a.mean(-1, keepdim=True), (a * h).mean(-1, keepdim=True)
    gx = r * (a - ma - h * mh)
    e_ma = (k + 2) * U * a.abs().mean(-1, keepdim=True)
    e_mh = (k + 3) * U * (a * h).abs().mean(-1, keepdim=True) + (a.abs() * e_h).mean(-1, keepdim=True)
    e_in = 4 * U * (a.abs() + ma.abs() + (h * mh).abs()) + e_ma + h.abs() * e_mh + e_h * mh.abs() + e_h * e_mh
    step = half_step(x.dtype)
    e_gx = (r + e_r) * e_in + e_r * (a - ma - h * mh).abs() + 3 * U * gx.abs()
    e_gx = e_gx * (1 + step) + step * gx.abs() + tiny(x.dtype)
    kr = x.shape[0] / 8 + 600  # a chain over part of the rows, and the joins of the parts
    gw, gb = (G * h).sum(0), G.sum(0)
    e_gw = (G.abs() * e_h).sum(0) + (kr + 2) * U * (G * h).abs().sum(0)
    e_gb = kr * U * G.abs().sum(0)
    return (y, gx, gw, gb), (e_y, e_gx, e_gw, e_gb)


LN_SHAPES = [(1, 1), (3, 2), (5, 7), (2, 32), (9, 33), (64, 384), (33, 512), (7, 515), (130, 1000), (17, 1024),
             (6, 1536), (5, 2047), (4, 4096), (3, 5001), (2, 8192), (2, 20000), (3, 13001), (1500, 96), (777, 130), (1, 384)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,D", LN_SHAPES)
@pytest.mark.parametrize("dtype", FLOATS)
def test_layer_norm_values_and_gradients(ops, rows, D, dtype):
    x, w, b, gy = ln_case(rows, D, dtype, rows * 7 + D, w_dtype=dtype if D % 2 else torch.float32)
    want, err = ln_exact(x, w, b, gy, 1e-5, dtype)
    xd, wd, bd = (t.to(DEV).requires_grad_(True) for t in (x, w, b))
    y = ops.layer_norm(xd, wd, bd, 1e-5)
    got = (y, *torch.autograd.grad(y, (xd, wd, bd), gy.to(DEV)))
    assert [t.dtype for t in got] == [dtype, dtype, w.dtype, w.dtype]
    for name, t, v, e in zip(("y", "gx", "gw", "gb"), got, want, err):
        if name in ("gw", "gb"):
            e = e + half_step(w.dtype) * (v.abs() + e) + tiny(w.dtype)
        assert_within(t, v, e, name)
    assert torch.equal(ops.layer_norm(xd.detach(), wd.detach(), bd.detach(), 1e-5), y)


@pytest.mark.gpu
@pytest.mark.parametrize("with_w,with_b", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16),
                                             (torch.float16, torch.bfloat16)])
def test_layer_norm_without_parameters_and_other_output_types(ops, with_w, with_b, dtype, out_dtype):
    x, w, b, gy = ln_case(37, 200, dtype, 3)
    gy = gy.to(out_dtype)
    w, b = w if with_w else None, b if with_b else None
    want, err = ln_exact(x, w, b, gy, 1e-5, out_dtype)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b) if t is not None]
    it = iter(leaves)
    args = [next(it) if t is not None else None for t in (x, w, b)]
    y = ops.layer_norm(*args, 1e-5, out_dtype=out_dtype)
    assert y.dtype == out_dtype
    grads = iter(torch.autograd.grad(y, leaves, gy.to(DEV)))
    assert_within(y, want[0], err[0], "y")
    for i, (t, name) in enumerate(zip((x, w, b), ("gx", "gw", "gb"))):
        if t is not None:
            assert_within(next(grads), want[1 + i], err[1 + i], name)


@pytest.mark.gpu
@pytest.mark.parametrize("start,D,pitch", [(0, 515, 643), (8, 384, 1152), (3, 64, 200), (1, 1001, 1003), (5, 32, 40)])
@pytest.mark.parametrize("dtype", FLOATS)
def test_layer_norm_reads_column_slices(ops, start, D, pitch, dtype):
    wide, w, b, _ = ln_case(21, pitch, dtype, start + D)
    wide, w, b = wide.to(DEV), w.to(DEV)[:D], b.to(DEV)[:D]
    gy = torch.randn(3, 7, D, generator=gen(1)).to(dtype).to(DEV)
    xs = wide.view(3, 7, pitch)[..., start:start + D]
    res = []
    for x in (xs.detach(), xs.contiguous()):
        x.requires_grad_(True)
        y = ops.layer_norm(x, w, b)
        res.append((y, *torch.autograd.grad(y, x, gy)))
    # aligned and unaligned rows may split a row's sums differently: two results, each within its bound
    want, err = ln_exact(xs.reshape(21, D).cpu(), w.cpu(), b.cpu(), gy.reshape(21, D).cpu(), 1e-5, dtype)
    for y, gx in res:
        assert y.is_contiguous() and gx.shape == (3, 7, D)
        assert_within(y.reshape(21, D), want[0], err[0], "y")
        assert_within(gx.reshape(21, D), want[1], err[1], "gx")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,D", [(1, 8), (2, 384), (147, 96), (148, 384), (149, 515), (1184, 64), (1185, 1000),
                                    (5000, 384), (3001, 2048), (700, 8192), (150, 20000), (70, 12801)])
@pytest.mark.parametrize("dtype", FLOATS)
def test_layer_norm_parameter_gradients_are_exact_on_integers(ops, rows, D, dtype):
    """With mean 0, 1/std 1 and small integers g_w = sum g x and g_b = sum g are
    exact in any order: a lost or doubled row shows.  Sums stay below 2^24."""
    g = gen(rows + D)
    x = torch.randint(-8, 9, (rows, D), generator=g).to(dtype)
    gy = torch.randint(-8, 9, (rows, D), generator=g).to(dtype)
    stats = torch.tensor([0.0, 1.0]).repeat(rows, 1).to(DEV)
    w = torch.ones(D, device=DEV)
    _, gw, gb = ops.layer_norm_bwd(gy.to(DEV), x.to(DEV), stats, w, need_x=False)
    assert torch.equal(gw.cpu().double(), (gy.double() * x.double()).sum(0))
    assert torch.equal(gb.cpu().double(), gy.double().sum(0))
    gx, gw2, gb2 = ops.layer_norm_bwd(gy.to(DEV), x.to(DEV), stats, w)
    assert torch.equal(gw, gw2) and torch.equal(gb, gb2) and gx.shape == x.shape


@pytest.mark.gpu
def test_layer_norm_large_offset_keeps_its_digits(ops):
    """x = 1000 + noise: var from squares of x itself would lose 20 of 24 bits."""
    x, w, b, gy = ln_case(50, 384, torch.float32, 5, offset=0.0)
    x = x + 1000.0
    want, err = ln_exact(x, w, b, gy, 1e-5, torch.float32)
    y = ops.layer_norm(x.to(DEV), w.to(DEV), b.to(DEV))
    assert_within(y, want[0], err[0], "y")
    # the bound itself: mean's error k u |x| times 1/std, about 28 * 6e-8 * 1000 / 1.5
    assert err[0].max() < 0.02


@pytest.mark.gpu
def test_layer_norm_constant_rows_nan_rows_and_empty_input(ops):
    x = torch.randn(6, 100, generator=gen(1))
    x[1] = 2.5
    x[3, 7] = float("nan")
    x[4, 9] = float("inf")
    w = torch.ones(100)
    y = ops.layer_norm(x.to(DEV), w.to(DEV), w.to(DEV)).cpu()
    assert torch.equal(y[1], torch.ones(100))  # x - mean is 0
    assert y[3].isnan().all() and y[4].isnan().all()
    for i in (0, 2, 5):
        assert torch.isfinite(y[i]).all()
    xe = torch.empty(0, 3, 100, device=DEV, requires_grad=True)
    wd = w.to(DEV).requires_grad_(True)
    ye = ops.layer_norm(xe, wd)
    gx, gw = torch.autograd.grad(ye, (xe, wd), torch.empty_like(ye))
    assert ye.shape == (0, 3, 100) and gx.shape == xe.shape and torch.equal(gw.cpu(), torch.zeros(100))


@pytest.mark.gpu
def test_layer_norm_gradient_against_differences(ops):
    """<gx, v> + <gw, vw> + <gb, vb> against the central difference of the 64-bit
    forward (step 1e-5: its own error is far below the bound's)."""
    x, w, b, gy = ln_case(9, 77, torch.float32, 11)
    vs = [torch.randn(t.shape, generator=gen(12 + i), dtype=torch.float64) for i, t in enumerate((x, w, b))]

    def f(s):
        X, W, Bv = (t.double() + s * v for t, v in zip((x, w, b), vs))
        c = X - X.mean(-1, keepdim=True)
        return ((c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5) * W + Bv) * gy.double()).sum()

    diff = (f(1e-5) - f(-1e-5)) / 2e-5
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(ops.layer_norm(*leaves), leaves, gy.to(DEV))
    _, err = ln_exact(x, w, b, gy, 1e-5, torch.float32)
    bound = sum((e * v.abs()).sum() for e, v in zip(err[1:], vs)) + 1e-7
    assert abs(sum((t.cpu().double() * v).sum() for t, v in zip(got, vs)) - diff) <= bound


# ------------------------------------------------------------------ embedding


EMB_SHAPES = [(1, 1, 1), (1, 5, 3), (64, 256, 384), (100, 7, 33), (513, 1000, 512), (4096, 256, 384), (2000, 3, 8),
              (3000, 40000, 24), (33, 2, 1030), (5000, 70000, 5), (257, 300, 2048), (9000, 1, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,V,D", EMB_SHAPES)
@pytest.mark.parametrize("dtype", FLOATS)
def test_embedding_forward_is_the_rounded_product(ops, n, V, D, dtype):
    g = gen(n + V + D)
    w = torch.randn(V, D, generator=g).to(dtype)
    tok = torch.randint(0, V, (n,), generator=g)
    scale = D ** 0.5
    out, bad = ops.embedding(tok.to(DEV), w.to(DEV), scale)
    assert int(bad) == 0 and out.dtype == dtype
    # one fp32 product and one rounding: equality
    assert torch.equal(out.cpu(), (w[tok].float() * torch.tensor(scale, dtype=torch.float32)).to(dtype))
    wide, _ = ops.embedding(tok.to(DEV), w.to(DEV), 1.0, out_dtype=torch.float32)
    assert torch.equal(wide.cpu(), w[tok].float())


def scatter_exact(tok, g, V, scale, padding_idx=None):
    out = torch.zeros(V, g.shape[-1], dtype=torch.float64)
    keep = (tok >= 0) & (tok < V)
    if padding_idx is not None:
        keep &= tok != padding_idx
    out.index_add_(0, tok[keep], g[keep].double())
    return out * scale


def token_mix(n, V, kind, g):
    if kind == "uniform":
        return torch.randint(0, V, (n,), generator=g)
    if kind == "one":  # every token the same
        return torch.full((n,), V - 1)
    if kind == "falling":
        return (torch.arange(n).flip(0) * V) // max(n, 1)
    tok = (torch.rand(n, generator=g) ** 4 * V).long().clamp(max=V - 1)  # long-tailed
    return torch.randperm(V, generator=g)[tok]


@pytest.mark.gpu
@pytest.mark.parametrize("n,V,D", EMB_SHAPES)
@pytest.mark.parametrize("kind", ["uniform", "one", "falling", "tail"])
def test_embedding_gradient_is_exact_on_integers(ops, n, V, D, kind):
    """Integers below 2^24 in the sums: equality in every type of g, whatever the
    order; a token's row that is lost, doubled or misplaced shows."""
    gr = gen(n * 3 + V + D)
    tok = token_mix(n, V, kind, gr)
    gi = torch.randint(-100, 101, (n, D), generator=gr)
    want = scatter_exact(tok, gi, V, 0.5)
    for dtype in FLOATS:
        got = ops.embedding_bwd(gi.to(dtype).to(DEV), tok.to(DEV), V, 0.5)
        assert got.dtype == torch.float32 and torch.equal(got.cpu().double(), want), dtype


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
def test_embedding_gradient_values(ops, dtype):
    """Real values: a row's sum over c tokens errs by at most (c + 2) u of its
    absolute sum (any order), times the scale's product, and half a step."""
    n, V, D = 6000, 501, 130
    gr = gen(4)
    tok = token_mix(n, V, "tail", gr)
    gy = torch.randn(n, D, generator=gr).to(dtype)
    w = torch.randn(V, D, generator=gr).to(dtype).to(DEV).requires_grad_(True)
    scale = D ** 0.5
    out, _ = ops.embedding(tok.to(DEV), w, scale)
    (got,) = torch.autograd.grad(out, w, gy.to(DEV))
    want = scatter_exact(tok, gy, V, scale)
    c = torch.bincount(tok, minlength=V).double().unsqueeze(1)
    e = (c + 4) * U * scatter_exact(tok, gy.abs(), V, scale)
    assert got.dtype == dtype
    assert_within(got, want, e * (1 + half_step(dtype)) + half_step(dtype) * want.abs() + tiny(dtype), "gw")
    again = torch.autograd.grad(ops.embedding(tok.to(DEV), w, scale)[0], w, gy.to(DEV))[0]
    assert torch.equal(got, again)  # fixed order of the sums


@pytest.mark.gpu
def test_embedding_gradient_against_differences(ops):
    """The operator is linear in the weight: the difference quotient is exact."""
    tok = torch.randint(0, 11, (4, 9), generator=gen(1))
    w = torch.randint(-5, 6, (11, 6), generator=gen(2)).float()
    gy = torch.randint(-5, 6, (4, 9, 6), generator=gen(3)).float()
    f = lambda m: ((m[tok] * 2.0) * gy).double().sum()  # noqa: E731
    wd = w.to(DEV).requires_grad_(True)
    (got,) = torch.autograd.grad(ops.embedding(tok.to(DEV), wd, 2.0)[0], wd, gy.to(DEV))
    for v, d in [(0, 0), (10, 5), (3, 2)]:
        step = torch.zeros_like(w)
        step[v, d] = 1.0
        assert float(got[v, d]) == float(f(w + step) - f(w))


@pytest.mark.gpu
def test_embedding_second_derivatives(ops):
    """The gradient is linear in g: its own gradient is the lookup, without the padding
    row (integers: equality with torch's)."""
    tok = torch.randint(0, 7, (5, 6), generator=gen(1)).to(DEV)
    w = torch.randint(-4, 5, (7, 12), generator=gen(2)).float().to(DEV).requires_grad_(True)
    v = torch.randint(-4, 5, (7, 12), generator=gen(3)).float().to(DEV)
    res = []
    for f in (lambda: ops.embedding(tok, w, 2.0, padding_idx=3)[0],
              lambda: torch.nn.functional.embedding(tok, w, padding_idx=3) * 2.0):
        (gw,) = torch.autograd.grad(f().pow(2).sum(), w, create_graph=True)
        (gg,) = torch.autograd.grad((gw * v).sum(), w)
        res.append((gw.detach(), gg))
    assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1])


@pytest.mark.gpu
def test_embedding_gradients_in_a_batch(ops):
    """``is_grads_batched``: each gradient of the batch is that of its own call (integers:
    equality), tokens outside the vocabulary and the padding row without one."""
    tok = torch.randint(0, 7, (5, 6), generator=gen(1))
    tok[0, 0], tok[1, 1] = -1, 1 << 40
    w = torch.randn(7, 12, generator=gen(2)).to(DEV).requires_grad_(True)
    g = torch.randint(-9, 10, (3, 5, 6, 12), generator=gen(3)).float().to(DEV)
    out, bad = ops.embedding(tok.to(DEV), w, 0.5, padding_idx=2)
    (got,) = torch.autograd.grad(out, w, g, is_grads_batched=True)
    for i in range(3):
        want = scatter_exact(tok.flatten(), g[i].reshape(30, 12).cpu(), 7, 0.5, 2)
        assert torch.equal(got[i].cpu().double(), want)


@pytest.mark.gpu
def test_embedding_launches_are_counted_and_recorded(ops):
    """A counter or recorder around both directions, one of them, or neither sees the
    launches inside it (lookup and sort, sums and join), with equal results."""
    tok = torch.randint(0, 50, (6, 40), generator=gen(1)).to(DEV)
    w = torch.randn(50, 24, generator=gen(2)).to(DEV).requires_grad_(True)
    g = torch.randn(6, 40, 24, generator=gen(3)).to(DEV)
    out, bad = ops.embedding(tok, w, 2.0)
    want = out, torch.autograd.grad(out, w, g)[0]
    for kind in (_lib.LaunchCounter, _lib.LaunchRecorder):
        def seen(c):
            return c.counts if kind is _lib.LaunchCounter else {k: v["launches"] for k, v in c.summary().items()}
        with kind() as both:
            out, bad = ops.embedding(tok, w, 2.0)
            (gw,) = torch.autograd.grad(out, w, g, retain_graph=True)
        with kind() as backward:
            (again,) = torch.autograd.grad(out, w, g)
        with kind() as forward:
            out2, _ = ops.embedding(tok, w, 2.0)
        (gw2,) = torch.autograd.grad(out2, w, g)
        assert seen(both) == {"embedding_fwd": 2, "embedding_bwd": 2}
        assert seen(backward) == {"embedding_bwd": 2} and seen(forward) == {"embedding_fwd": 2}
        for t, v in ((out, want[0]), (out2, want[0]), (gw, want[1]), (again, want[1]), (gw2, want[1])):
            assert torch.equal(t, v)
        assert int(bad) == 0


@pytest.mark.gpu
def test_embedding_node_keeps_to_torchs_rules(ops):
    """A second backward needs retain_graph, tokens changed in place after the lookup are
    an error, an unused result has no gradient, and a row-strided, transposed or empty
    weight or token tensor is read as it is."""
    tok = torch.randint(0, 9, (20,), generator=gen(1)).to(DEV)
    w = torch.randn(9, 16, generator=gen(2)).to(DEV).requires_grad_(True)
    out, _ = ops.embedding(tok, w)
    out.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        out.sum().backward()
    counts = torch.bincount(tok, minlength=9).float().unsqueeze(1).expand(9, 16)
    assert torch.equal(w.grad, counts)
    out, _ = ops.embedding(tok, w)
    tok2 = tok.clone()
    out2, _ = ops.embedding(tok2, w)
    tok2 += 1
    with pytest.raises(RuntimeError, match="inplace|in-place"):
        out2.sum().backward()
    assert torch.autograd.grad((out * 0 + w.sum()).sum(), w)[0].eq(320).all()
    for leaf in (torch.randn(9, 40, generator=gen(3))[:, 3:19], torch.randn(16, 9, generator=gen(4)).t()):
        leaf = leaf.to(DEV).detach()
        base = leaf.clone(memory_format=torch.contiguous_format)
        leaf.requires_grad_(True)
        out, _ = ops.embedding(tok, leaf, 0.5)
        (gw,) = torch.autograd.grad(out.sum(), leaf)
        assert torch.equal(out, base[tok] * 0.5) and torch.equal(gw, counts * 0.5)
    for dt in FLOATS:
        out, _ = ops.embedding(tok, w, 3.0, out_dtype=dt)
        (gw,) = torch.autograd.grad(out, w, torch.ones_like(out))
        assert out.dtype == dt and gw.dtype == torch.float32 and torch.equal(gw, counts * 3)
    with pytest.raises(TypeError):
        ops.embedding(tok, w, watch=1)


@pytest.mark.gpu
@pytest.mark.parametrize("n,V,D", [(50, 9, 24), (3000, 257, 40)])
def test_embedding_padding_and_bad_tokens(ops, n, V, D):
    gr = gen(n)
    tok = torch.randint(0, V, (n,), generator=gr)
    tok[::7] = 2
    gi = torch.randint(-50, 51, (n, D), generator=gr).float()
    w = torch.randn(V, D, generator=gr).to(DEV).requires_grad_(True)
    out, bad = ops.embedding(tok.to(DEV), w, 1.0, padding_idx=2)
    (got,) = torch.autograd.grad(out, w, gi.to(DEV))
    assert int(bad) == 0 and torch.equal(out.cpu(), w.detach().cpu()[tok])  # the row itself is read as it is
    assert torch.equal(got.cpu().double(), scatter_exact(tok, gi, V, 1.0, 2)) and not got[2].any()
    for wrong in (-1, V, -(1 << 40), 1 << 40, (1 << 32) + 1):
        t = tok.clone()
        t[n // 2] = wrong
        out, bad = ops.embedding(t.to(DEV), w, 1.0)
        (got,) = torch.autograd.grad(out, w, gi.to(DEV))
        assert int(bad) == 1 and not out[n // 2].any()
        assert torch.equal(got.cpu().double(), scatter_exact(t, gi, V, 1.0))


@pytest.mark.gpu
def test_embedding_token_types_layouts_and_empty_input(ops):
    V, D = 50, 24
    wide = torch.randn(V, 64, generator=gen(1)).to(DEV)
    w = wide[:, 8:8 + D]
    tok = torch.randint(0, V, (6, 10), generator=gen(2)).to(DEV)
    want = w[tok]
    for t in (tok, tok.int(), tok.to(torch.int16), tok.to(torch.uint8), tok.t().contiguous().t()):
        assert torch.equal(ops.embedding(t, w)[0], want)
    assert torch.equal(ops.embedding(tok[:, ::2], w)[0], want[:, ::2])
    assert torch.equal(ops.embedding(tok[0, 0], w)[0], want[0, 0])
    # a gradient that is one value expanded, and one with transposed storage
    wl = w.detach().requires_grad_(True)
    (g1,) = torch.autograd.grad(ops.embedding(tok, wl)[0].sum(), wl)
    assert torch.equal(g1, torch.bincount(tok.flatten(), minlength=V).float().unsqueeze(1).expand(V, D))
    gt = torch.randint(-9, 10, (D, 10, 6), generator=gen(3)).float().to(DEV)
    (g2,) = torch.autograd.grad(ops.embedding(tok, wl)[0], wl, gt.permute(2, 1, 0))
    assert torch.equal(g2.cpu().double(), scatter_exact(tok.flatten().cpu(), gt.permute(2, 1, 0).reshape(60, D).cpu(),
                                                        V, 1.0))
    empty = torch.empty(0, 3, dtype=torch.int64, device=DEV)
    out, bad = ops.embedding(empty, wl)
    (g3,) = torch.autograd.grad(out, wl, torch.empty_like(out))
    assert out.shape == (0, 3, D) and int(bad) == 0 and not g3.any()


SORT_TWICE = """
import torch
from spikingtransformer_b200 import ops
g = torch.Generator().manual_seed(1)
n, V, D = 40000, 5000, 24
tok = torch.randint(0, V, (n,), generator=g)
gi = torch.randint(-9, 10, (n, D), generator=g).float()
want = torch.zeros(V, D).index_add_(0, tok, gi)
w = torch.zeros(V, D, device="cuda", requires_grad=True)
out, _ = ops.embedding(tok.cuda(), w)
got = [torch.autograd.grad(out, w, gi.cuda())[0], ops.embedding_bwd(gi.cuda(), tok.cuda(), V)]
assert all(torch.equal(t.cpu(), want) for t in got)
"""


@pytest.mark.gpu
@pytest.mark.parametrize("largest", ["8", "16"])
def test_embedding_sorts_without_the_largest_clusters(largest):
    """A device that holds no cluster of 16 blocks sorts many tokens with 8."""
    import os
    import subprocess
    import sys
    env = dict(os.environ, SPK_SORT_CLUSTER=largest)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", SORT_TWICE], cwd=root, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


# ------------------------------------------------------------------ token log probabilities


def lp_exact(logits, tok, K, ignore=-100):
    """Values and bounds in 64 bits.  Terms of a bound: the T-mean rounded once and
    the constant log2 e (relative u each, on z), the rounding of t = z log2 e - c
    (u |t|), 2^t (2^-22 relative), sums in chains of k, and the last few steps."""
    z = logits.double().mean(0).float().double()  # the operator's mean is rounded once to fp32
    V = z.shape[-1]
    k = V / 128 + 64
    zm = torch.where(torch.isinf(z), 0.0, z).abs().amax(-1)
    lse = torch.logsumexp(z, -1)
    lp = z - lse.unsqueeze(-1)
    p = lp.exp()
    lpf = torch.where(p > 0, lp, 0.0)
    H = -(p * lpf).sum(-1)
    t = lpf.abs() + (z.amax(-1, keepdim=True) - lse.unsqueeze(-1)).abs() + 1  # at least |t_j| ln 2
    mt, mt2 = (p * t).sum(-1), (p * t * t).sum(-1)
    e_lse = 4 * U * zm + (k + 10) * U + 2.0 ** -22 + 2 * U * mt
    e_lp = (e_lse.unsqueeze(-1) + 4 * U * zm.unsqueeze(-1) + 6 * U * t)
    e_H = 2 * e_lse + ((k + 10) * U + 2.0 ** -22) * (1 + mt) + 2 * U * mt2 + 8 * U * (mt + H.abs() + 1) \
        + 8 * U * zm * (1 + mt)
    used = (tok != ignore) & (tok >= 0) & (tok < V)
    y = tok.clamp(0, V - 1).unsqueeze(-1)
    out = {"z": z, "p": p, "lp": lp, "lpf": lpf, "H": H, "e_lp": e_lp, "e_H": e_H, "used": used, "y": y,
           "logp": torch.where(used, lp.gather(-1, y).squeeze(-1), 0.0), "entropy": torch.where(used, H, 0.0),
           "e_logp": e_lp.gather(-1, y).squeeze(-1)}
    if K:
        idx = torch.sort(z, dim=-1, descending=True, stable=True).indices[..., :K]
        out["top_idx"] = torch.where(used.unsqueeze(-1), idx, -1)
        out["top_logp"] = torch.where(used.unsqueeze(-1), lp.gather(-1, idx), 0.0)
        out["e_top"] = e_lp.gather(-1, idx)
    return out


def lp_grad_exact(o, gl, gh, gt, T, dtype):
    """dlogits of one step and its bound."""
    used = o["used"].double()
    gl = torch.zeros_like(used) if gl is None else gl.double() * used
    gh = torch.zeros_like(used) if gh is None else gh.double() * used
    G = gl.clone()
    if gt is not None:
        G = G + (gt.double() * used.unsqueeze(-1)).sum(-1)
    u1 = lambda v: v.unsqueeze(-1)  # noqa: E731
    F = u1(G) + u1(gh) * (o["lpf"] + u1(o["H"]))
    d = -o["p"] * F
    hot = torch.zeros_like(d)
    hot.scatter_add_(-1, o["y"], u1(gl))
    n_top = 0
    mag = hot.abs()
    if gt is not None:
        n_top = gt.shape[-1]
        add = gt.double() * u1(used)
        hot.scatter_add_(-1, o["top_idx"].clamp(min=0), add)
        mag.scatter_add_(-1, o["top_idx"].clamp(min=0), add.abs())
    Gm = u1(gl.abs() + (0 if gt is None else (gt.double() * u1(used)).abs().sum(-1)))
    e_F = u1(gh.abs()) * (o["e_lp"] + u1(o["e_H"])) + (n_top + 6) * U * (Gm + u1(gh.abs()) * (o["lpf"].abs()
                                                                                         + u1(o["H"]) + 2))
    e = o["p"] * (e_F + F.abs() * (o["e_lp"] + 2.0 ** -22 + 6 * U)) + 4 * U * (mag + d.abs())
    d, e = (d + hot) / T, e / T
    return d, e * (1 + half_step(dtype)) + (half_step(dtype) + U) * d.abs() + tiny(dtype) + 2.0 ** -120


LP_SHAPES = [(1, 1, 1), (1, 3, 2), (4, 5, 31), (1, 9, 32), (3, 7, 33), (4, 130, 256), (10, 33, 1000), (1, 17, 1023),
             (2, 5, 2048), (1, 6, 2049), (1, 4, 4097), (4, 3, 8200), (1, 3, 50001), (1, 1, 131072), (1, 600, 96)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,rows,V", LP_SHAPES)
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("K", [0, 5, 32])
def test_token_logprobs_values_and_gradients(ops, T, rows, V, dtype, K):
    K = min(K, V)
    g = gen(T + rows + V)
    x = (torch.randn(T, rows, V, generator=g) * 3).to(dtype)
    tok = torch.randint(0, V, (rows,), generator=g)
    if rows > 3:
        tok[1] = -100
    o = lp_exact(x, tok, K)
    xd = x.to(DEV).requires_grad_(True)
    logp, H, top, idx, bad = ops.token_logprobs(xd, tok.to(DEV), top_k=K)
    assert int(bad) == 0 and logp.dtype == torch.float32
    assert_within(logp, o["logp"], o["e_logp"], "logp")
    assert_within(H, o["entropy"], o["e_H"], "entropy")
    gs = [torch.randn(rows, generator=g), torch.randn(rows, generator=g)]
    outs = [logp, H]
    if K:
        assert torch.equal(idx.cpu(), o["top_idx"])
        assert_within(top, o["top_logp"], o["e_top"], "top_logp")
        gs.append(torch.randn(rows, K, generator=g))
        outs.append(top)
    else:
        assert top is None and idx is None
    (gx,) = torch.autograd.grad(outs, xd, [t.to(DEV) for t in gs], retain_graph=True)
    d, e = lp_grad_exact(o, gs[0], gs[1], gs[2] if K else None, T, dtype)
    for t in range(T):
        assert_within(gx[t], d, e, "grad")
    # each output alone
    (gx,) = torch.autograd.grad(logp, xd, gs[0].to(DEV), retain_graph=True)
    assert_within(gx[0], *lp_grad_exact(o, gs[0], None, None, T, dtype), "grad of logp")
    (gx,) = torch.autograd.grad(H, xd, gs[1].to(DEV), retain_graph=True)
    assert_within(gx[T - 1], *lp_grad_exact(o, None, gs[1], None, T, dtype), "grad of entropy")
    if K:
        (gx,) = torch.autograd.grad(top, xd, gs[2].to(DEV))
        assert_within(gx[0], *lp_grad_exact(o, None, None, gs[2], T, dtype), "grad of top_logp")
    with torch.no_grad():
        again = ops.token_logprobs(xd, tok.to(DEV), top_k=K)
    assert all(a is b or torch.equal(a, b) for a, b in zip(again, (logp, H, top, idx, bad)))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [8, 300, 5000, 40000])
@pytest.mark.parametrize("order", ["equal", "rising", "falling", "few values", "zeros of both signs"])
def test_top_alternatives_take_the_lower_index_on_ties(ops, V, order):
    rows, K = 6, 8
    if order == "equal":
        x = torch.full((1, rows, V), 0.25)
    elif order == "rising":
        x = (torch.arange(V) / V).expand(1, rows, V).contiguous()
    elif order == "falling":
        x = (-torch.arange(V) / V).expand(1, rows, V).contiguous()
    elif order == "few values":
        x = torch.randint(0, 3, (1, rows, V), generator=gen(V)).float()
    else:
        x = torch.zeros(1, rows, V) * torch.where(torch.arange(V) % 2 == 0, -1.0, 1.0)
    tok = torch.zeros(rows, dtype=torch.int64)
    o = lp_exact(x, tok, K)
    _, H, top, idx, _ = ops.token_logprobs(x.to(DEV), tok.to(DEV), top_k=K)
    assert torch.equal(idx.cpu(), o["top_idx"])
    assert_within(top, o["top_logp"], o["e_top"], "top_logp")
    assert_within(H, o["entropy"], o["e_H"], "entropy")


@pytest.mark.gpu
def test_near_ties_of_the_step_mean_keep_the_exact_order(ops):
    """fp32 logits of 4 steps whose means differ by a few units in the last place:
    the order is that of the means rounded once."""
    g = gen(3)
    base = torch.randn(4, 50, 1, generator=g)
    x = base + torch.randint(-3, 4, (4, 50, 256), generator=g) * 2.0 ** -23
    tok = torch.zeros(50, dtype=torch.int64)
    _, _, _, idx, _ = ops.token_logprobs(x.to(DEV), tok.to(DEV), top_k=16)
    assert torch.equal(idx.cpu(), lp_exact(x, tok, 16)["top_idx"])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 4, 5, 6, 7, 10, 12, 31])
def test_means_half_way_between_two_numbers_go_to_the_even_one(ops, T):
    """Sums of T steps whose quotient lies exactly half way (integers N = T (2 k + 1), k
    near 2^23 so that fp32 holds only every second of the quotients): with 1 / T
    rounded, an unguarded quotient falls to either side.  Neighbours differ by one
    such half step, so a wrong one shows in the order."""
    g = gen(T)
    V, rows = 64, 40
    means = (1 << 24) + torch.randint(0, 1 << 10, (rows, V), generator=g)  # odd ones: half way
    parts = torch.randint(-(1 << 20), 1 << 20, (T, rows, V), generator=g) * 2
    parts[-1] = 0
    parts[-1] = means * T - parts.sum(0)
    x = parts.float()
    # the last step in two, where fp32 does not hold it: what is left over goes to the first
    x[0] = x[0] + (parts[-1] - x[-1].long()).float()
    assert torch.equal(x.double().sum(0), (means * T).double())
    tok = torch.zeros(rows, dtype=torch.int64)
    want = torch.sort(x.double().mean(0).float(), dim=-1, descending=True, stable=True).indices[:, :32]
    _, _, _, idx, _ = ops.token_logprobs(x.to(DEV), tok.to(DEV), top_k=32)
    assert torch.equal(idx.cpu(), want)
    negative = torch.sort((-x).double().mean(0).float(), dim=-1, descending=True, stable=True).indices[:, :32]
    assert torch.equal(ops.token_logprobs(-x.to(DEV), tok.to(DEV), top_k=32)[3].cpu(), negative)


@pytest.mark.gpu
@pytest.mark.parametrize("T,V", [(1, 40), (4, 300), (1, 70000)])
@pytest.mark.parametrize("dtype", FLOATS)
def test_barred_symbols_and_rows_without_a_distribution(ops, T, V, dtype):
    rows, K = 8, 6
    g = gen(V)
    x = (torch.randn(T, rows, V, generator=g) * 2).to(dtype)
    x[:, :, torch.rand(V, generator=g) < 0.5] = float("-inf")
    x[:, :, 3] = 1.0
    x[:, 2, 4:] = float("-inf")                      # fewer symbols left than alternatives asked for
    x[:, 2, :3] = torch.tensor([0.5, float("-inf"), 0.25]).to(dtype)
    x[:, 3, :] = torch.finfo(dtype).min              # the type's lowest value everywhere: uniform
    x[0, 4, :] = float("-inf")                       # nothing left
    x[0, 5, V - 1] = float("nan")
    x[0, 6, 1] = float("inf")
    tok = torch.full((rows,), 3)
    tok[7] = -100
    gl, gh = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    o = lp_exact(x, tok, K)
    xd = x.to(DEV).requires_grad_(True)
    logp, H, top, idx, bad = ops.token_logprobs(xd, tok.to(DEV), top_k=K)
    (gx,) = torch.autograd.grad((logp, H), xd, (gl.to(DEV), gh.to(DEV)))
    d, e = lp_grad_exact(o, gl, gh, None, T, dtype)
    assert int(bad) == 0
    for r in (0, 1, 2, 7):
        assert_within(logp[r], o["logp"][r], o["e_logp"][r], "logp %d" % r)
        assert_within(H[r], o["entropy"][r], o["e_H"][r], "entropy %d" % r)
        assert torch.equal(idx[r].cpu(), o["top_idx"][r])
        fin = torch.isfinite(o["top_logp"][r])
        assert torch.equal(top[r].cpu()[~fin].double(), o["top_logp"][r][~fin])
        assert_within(top[r].cpu()[fin], o["top_logp"][r][fin], o["e_top"][r][fin], "top %d" % r)
        for t in range(T):
            assert_within(gx[t, r], d[r], e[r], "grad %d" % r)
    # all equal: logp = -log V, H = log V, whatever the common value
    lv = torch.tensor(float(V), dtype=torch.float64).log()
    k = (V / 128 + 80) * U + 2.0 ** -22
    logp, H = logp.detach(), H.detach()
    assert abs(float(logp[3]) + lv) <= k + 4 * U * lv and abs(float(H[3]) - lv) <= 2 * k + 8 * U * lv
    assert torch.equal(idx[3].cpu(), torch.arange(K))
    for r in (4, 5, 6):
        assert logp[r].isnan() and H[r].isnan() and top[r].isnan().all() and gx[:, r].isnan().all()
        assert len(set(idx[r].tolist())) == K and 0 <= int(idx[r].min()) and int(idx[r].max()) < V
    assert not gx[:, 7].any()


@pytest.mark.gpu
@pytest.mark.parametrize("T,rows,V", [(1, 9, 200), (2, 9, 1000), (1, 9, 1000), (1, 2400, 1000), (1, 9, 9000),
                                      (1, 300, 20000), (1, 9, 70000), (3, 9, 70001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [5, 32])
def test_alternatives_of_rows_with_more_nans_than_numbers(ops, T, rows, V, dtype, K):
    """Fewer numbers than alternatives asked for, more NaNs than are gathered at once: the
    numbers come first, then -inf, then NaNs, each by index, and nothing outside the row
    is read or written."""
    x = torch.full((rows, V), float("nan"))
    places = torch.randperm(V, generator=gen(V))[:K - 1]
    kinds = rows // 3  # a third all NaN, a third with K - 1 numbers, a third with -inf besides
    x[kinds:, places] = torch.arange(K - 1).float()
    x[2 * kinds:, places[:2]] = float("-inf")
    want = []
    for r in range(rows):
        key = x[r].clone()
        low = key == float("-inf")
        key[low] = -1.0
        key[key.isnan()] = -2.0
        want.append(torch.sort(key, descending=True, stable=True).indices[:K])
    xd = x.to(dtype).expand(T, rows, V).contiguous().to(DEV).requires_grad_(True)
    tok = torch.zeros(rows, dtype=torch.int64, device=DEV)
    logp, H, top, idx, bad = ops.token_logprobs(xd, tok, top_k=K)
    assert torch.equal(idx.cpu(), torch.stack(want)) and int(bad) == 0
    assert logp.isnan().all() and H.isnan().all() and top.isnan().all()
    (gx,) = torch.autograd.grad(top, xd, torch.ones_like(top))
    assert gx.isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [40, 300, 5000, 5001])
def test_infinities_among_the_steps(ops, V):
    """The mean over the steps where some are not finite, or their partial sums are not:
    -inf in the first, a later or every step bars the symbol, steps of +-3e38 whose
    mean is finite do not, +inf, NaN or both infinities take the row."""
    T, rows, K = 3, 10, 4
    x = torch.randn(T, rows, V, generator=gen(V))
    inf = float("inf")
    for c, steps in enumerate([(-inf, 1.0, 2.0), (1.0, -inf, 2.0), (1.0, 2.0, -inf), (-inf,) * 3, (-inf, -3e38, -3e38),
                               (-3e38, -3e38, -inf), (3e38, 3e38, -inf), (3e38, 3e38, -3e38 * 2 + 3.4e38),
                               (3.25, -3e38, 3e38)]):
        x[:, :, 5 + c] = torch.tensor(steps)[:, None]
    x[:, 0:6, 12] = 0.0  # the rows whose symbols are all of ordinary size but the barred ones
    x[1, 1, 30] = inf
    x[:, 2, 30] = torch.tensor([inf, -inf, 0.0])
    x[:, 3, 30] = torch.tensor([-inf, 0.0, inf])
    x[2, 4, 30] = float("nan")
    x[:, 5, 30] = torch.tensor([float("nan"), -inf, 0.0])
    tok = torch.zeros(rows, dtype=torch.int64)
    z = x.double().mean(0)
    z[:, 13] = 3.25 / 3  # 64 bits lose the 3.25 beside 3e38
    o = lp_exact(z.float()[None], tok, K)
    xd = x.to(DEV).requires_grad_(True)
    logp, H, top, idx, _ = ops.token_logprobs(xd, tok.to(DEV), top_k=K)
    gl = torch.randn(rows, generator=gen(1))
    (gx,) = torch.autograd.grad(logp, xd, gl.to(DEV))
    d, e = lp_grad_exact(o, gl, None, None, T, torch.float32)
    for r in range(1, 6):
        assert logp[r].isnan() and H[r].isnan() and gx[:, r].isnan().all()
    for r in (0, 6, 7, 8, 9):
        assert torch.equal(idx[r].cpu(), o["top_idx"][r])
        if r == 0:
            assert_within(logp[r], o["logp"][r], o["e_logp"][r], "logp")
            assert_within(H[r], o["entropy"][r], o["e_H"][r], "entropy")
            assert_within(gx[0, r], d[r], e[r], "grad")
        else:  # one symbol near 1e38 takes it all
            assert float(top[r, 0]) == 0 and int(idx[r, 0]) == 12 and float(H[r]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("V", [48, 300, 9000])
@pytest.mark.parametrize("dtype", FLOATS)
def test_lowest_values_are_above_minus_infinity(ops, V, dtype):
    """Rows with the type's lowest value at every third symbol and -inf elsewhere: the
    former share the probability, the latter have none."""
    rows = 4
    x = torch.full((1, rows, V), float("-inf"))
    x[:, :, ::3] = torch.finfo(dtype).min
    x[:, 1, 3] = 0.0  # one symbol above them takes it all
    tok = torch.tensor([0, 3, 1, 0])
    xd = x.to(dtype).to(DEV).requires_grad_(True)
    logp, H, top, idx, _ = ops.token_logprobs(xd, tok.to(DEV), top_k=2)
    (gx,) = torch.autograd.grad(logp[0] + H[3], xd)
    n = (V + 2) // 3
    ln = torch.tensor(float(n), dtype=torch.float64).log()
    tol = (V / 128 + 80) * U + 2.0 ** -22 + 8 * U * ln
    logp, H, top = (t.detach().double().cpu() for t in (logp, H, top))
    assert abs(logp[0] + ln) <= tol and abs(H[0] - ln) <= 2 * tol
    assert logp[1] == 0 and H[1] == 0 and idx[1, 0] == 3 and idx[1, 1] == 0
    assert logp[2] == float("-inf") and abs(H[2] - ln) <= 2 * tol
    assert idx[0].tolist() == [0, 3] and ((top[0] + ln).abs() <= tol).all()
    want = torch.zeros(V, dtype=torch.float64)
    want[::3] = -1.0 / n
    want[0] += 1.0
    assert_within(gx[0, 0], want, (tol + half_step(dtype)) * want.abs() + tol / n + tiny(dtype), "grad")
    # entropy's gradient -p (log p + H) is 0 where all are alike: the error of log p + H
    assert gx[0, 3].abs().max() <= 4 * tol / n and not gx[0, 2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("T,V", [(1, 1), (1, 40), (3, 300), (1, 5000), (1, 70000)])
@pytest.mark.parametrize("dtype", FLOATS)
def test_rows_of_one_symbol_have_no_positive_logp_and_no_negative_entropy(ops, T, V, dtype):
    """One symbol with (nearly) all of the probability, at maxima of any size: logp <= 0
    and entropy >= 0, both within their bounds of the exact values near 0."""
    rows, K = 64, min(2, V)
    g = gen(V)
    x = torch.full((T, rows, V), float("-inf"))
    tok = torch.randint(0, V, (rows,), generator=g)
    if V > 1:
        x[:, rows // 2:] = -20.0 + torch.rand(T, rows // 2, V, generator=g)  # half: others far below
    x[:, torch.arange(rows), tok] = torch.randn(T, rows, generator=g) * 10 + 20
    x = x.to(dtype)
    o = lp_exact(x, tok, K)
    xd = x.to(DEV).requires_grad_(True)
    logp, H, top, idx, _ = ops.token_logprobs(xd, tok.to(DEV), top_k=K)
    assert (logp <= 0).all() and (H >= 0).all() and (top <= 0).all()
    assert torch.equal(idx[:, 0].cpu(), tok)
    assert_within(logp, o["logp"], o["e_logp"], "logp")
    assert_within(H, o["entropy"], o["e_H"], "entropy")
    gl, gh = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    (gx,) = torch.autograd.grad((logp, H), xd, (gl.to(DEV), gh.to(DEV)))
    assert_within(gx[0], *lp_grad_exact(o, gl, gh, None, T, dtype), "grad")


@pytest.mark.gpu
def test_token_logprobs_near_one_keeps_its_digits(ops):
    """p_y = 1 - 1e-7 or so: logp comes from t_y - log2 S, not from the difference
    of two numbers near 20."""
    x = torch.zeros(1, 4, 64)
    x[:, :, 5] = torch.tensor([16.0, 18.0, 20.0, 24.0])
    tok = torch.full((4,), 5)
    logp = ops.token_logprobs(x.to(DEV), tok.to(DEV))[0].cpu().double()
    want = x.double().log_softmax(-1)[0, :, 5]
    # S = 1 + s with t_y exact to u |t_y|, |t_y| <= 1/2 ... and log2 S exact to a few u
    assert ((logp - want).abs() <= 8 * U).all()


@pytest.mark.gpu
def test_token_logprobs_layouts_bad_tokens_and_empty_input(ops):
    g = gen(9)
    T, B, N, V = 4, 3, 6, 70
    x = torch.randn(T, B, N, V, generator=g).to(DEV)
    tok = torch.randint(0, V, (B, N), generator=g).to(DEV)
    full = ops.token_logprobs(x, tok, top_k=3)
    last = ops.token_logprobs(x[:, :, -1], tok[:, -1], top_k=3)          # rows of a decoding step
    cut = ops.token_logprobs(x[:, 1:, :, :], tok[1:], top_k=3)
    perm = ops.token_logprobs(x.transpose(1, 2), tok.t(), top_k=3)       # not collapsible: copied
    narrow = ops.token_logprobs(torch.cat([x, x], -1)[..., 1:1 + V], tok, top_k=3)
    odd = ops.token_logprobs(x[..., 1:], tok.clamp(max=V - 2), top_k=3)
    same = ops.token_logprobs(x[..., 1:].contiguous(), tok.clamp(max=V - 2), top_k=3)
    steps = ops.token_logprobs(x[:1].expand(T, B, N, V), tok, top_k=3)   # one step repeated is its own mean
    one = ops.token_logprobs(x[:1], tok, top_k=3)
    scalar = ops.token_logprobs(x[:, 0, 0], tok[0, 0], top_k=3)
    tol = dict(rtol=0, atol=1e-5)  # 16 u of values below 10, where aligned and unaligned rows split sums differently
    for i in range(4):
        for a, b in [(last[i], full[i][:, -1]), (cut[i], full[i][1:]), (perm[i], full[i].transpose(0, 1)),
                     (odd[i], same[i]), (steps[i], one[i]), (scalar[i], full[i][0, 0])]:
            assert torch.equal(a, b) if i == 3 else torch.allclose(a, b, **tol)
    assert torch.isfinite(narrow[0]).all()
    xl = x.detach().requires_grad_(True)
    (g1,) = torch.autograd.grad(ops.token_logprobs(xl[:, :, -1], tok[:, -1])[0].sum(), xl)
    (g2,) = torch.autograd.grad((xl.mean(0).log_softmax(-1)[:, -1]).gather(-1, tok[:, -1:]).sum(), xl)
    assert torch.allclose(g1, g2, rtol=0, atol=1e-6)
    for wrong in (-1, V, 1 << 40):
        t = tok.clone()
        t[1, 2] = wrong
        xl = x.detach().requires_grad_(True)
        logp, H, top, idx, bad = ops.token_logprobs(xl, t, top_k=2)
        (gx,) = torch.autograd.grad(logp.sum() + H.sum() + top.sum(), xl)
        logp, H = logp.detach(), H.detach()
        assert int(bad) == 1 and float(logp[1, 2]) == 0 and float(H[1, 2]) == 0
        assert (idx[1, 2] == -1).all() and not gx[:, 1, 2].any() and torch.isfinite(gx).all()
        assert torch.equal(logp[0], full[0][0])
    e = ops.token_logprobs(x[:, :0].detach().requires_grad_(True), tok[:0], top_k=2)
    assert e[0].shape == (0, N) and e[2].shape == (0, N, 2) and int(e[4]) == 0


@pytest.mark.gpu
def test_token_logprobs_gradient_against_differences(ops):
    g = gen(5)
    x = torch.randn(3, 7, 50, generator=g)
    tok = torch.randint(0, 50, (7,), generator=g)
    gl, gh, gt = (torch.randn(*s, generator=g) for s in ((7,), (7,), (7, 2)))
    v = torch.randn(3, 7, 50, generator=g, dtype=torch.float64)
    o = lp_exact(x, tok, 2)

    def f(s):
        lp = (x.double() + s * v).mean(0).log_softmax(-1)
        H = -(lp.exp() * lp).sum(-1)
        return ((lp.gather(-1, tok[:, None])[:, 0] * gl).sum() + (H * gh).sum()
                + (lp.gather(-1, o["top_idx"]) * gt).sum())

    diff = (f(1e-5) - f(-1e-5)) / 2e-5
    xd = x.to(DEV).requires_grad_(True)
    logp, H, top, _, _ = ops.token_logprobs(xd, tok.to(DEV), top_k=2)
    (gx,) = torch.autograd.grad((logp, H, top), xd, (gl.to(DEV), gh.to(DEV), gt.to(DEV)))
    d, e = lp_grad_exact(o, gl, gh, gt, 3, torch.float32)
    # the difference is of unrounded means: u |z| more on each logit
    bound = ((e + 4 * U * (d.abs() + o["p"])) * v.abs().sum(0)).sum() + 1e-6
    assert abs((gx.cpu().double() * v).sum() - diff) <= bound


@pytest.mark.gpu
def test_steps_up_to_those_of_a_lif(ops):
    """64 steps give the mean's values; 65 are refused, as by the LIF."""
    x = torch.randn(65, 3, 40, generator=gen(1))
    tok = torch.tensor([0, 39, 7])
    o = lp_exact(x[:64], tok, 0)
    logp, H = ops.token_logprobs(x[:64].to(DEV), tok.to(DEV))[:2]
    assert_within(logp, o["logp"], o["e_logp"], "logp")
    assert_within(H, o["entropy"], o["e_H"], "entropy")
    with pytest.raises(ValueError, match="64 steps"):
        ops.token_logprobs(x.to(DEV), tok.to(DEV))
    one = torch.ones(1, device=DEV)
    with pytest.raises(RuntimeError, match="64"):
        ops.lif_fwd(x.to(DEV), one, one, one)


# ------------------------------------------------------------------ in the model


def small_model(dropout=0.0):
    from spikingtransformer_b200.Seq2Seq import Seq2Seq
    torch.manual_seed(3)
    return Seq2Seq(patch_size=16, d_model=64, n_heads=4, ff_dim=128, num_encoder_layers=1, num_decoder_layers=1,
                   dropout=dropout, tgt_vocab_size=64, n_steps=4, image_encoder="patch").to(DEV)


@pytest.mark.gpu
def test_token_embedding_module_matches_the_lookup(ops):
    from spikingtransformer_b200.Seq2Seq import TokenEmbedding
    torch.manual_seed(1)
    m = TokenEmbedding(50, 96).to(DEV)
    tok = torch.randint(0, 50, (4, 17), device=DEV)
    g = torch.randint(-5, 6, (4, 17, 96), device=DEV).float()
    out = m(tok)
    (gw,) = torch.autograd.grad(out, m.embedding.weight, g)
    ref = m.embedding(tok) * 96 ** 0.5
    (rw,) = torch.autograd.grad(ref, m.embedding.weight, g)
    assert torch.equal(out, ref) and int(m.bad_tokens) == 0   # the product is rounded once on both sides
    # 68 tokens: each way sums a row's few terms (one scales before, one after) within (c + 2) u of their size
    size = torch.zeros(50, 96, device=DEV).index_add_(0, tok.flatten(), g.abs().flatten(0, 1)) * 96 ** 0.5
    assert ((gw - rw).abs() <= 2 * (68 + 2) * U * size).all()
    assert torch.equal(m(tok.int()), ref) and torch.equal(m(tok.float()), ref)
    seen = []
    hook = m.embedding.register_forward_hook(lambda *a: seen.append(1))
    assert torch.equal(m(tok), ref) and seen
    hook.remove()
    assert torch.equal(m.half()(tok), (m.embedding.weight[tok].float() * 96 ** 0.5).half())
    m.float().embedding.padding_idx = 3
    (gw,) = torch.autograd.grad(m(tok), m.embedding.weight, g)
    assert not gw[3].any()
    assert list(m.state_dict()) == ["embedding.weight"]
    m(tok + 50)
    assert int(m.bad_tokens) == 1


class CountedEmbedding(torch.nn.Embedding):
    """A forward of its own: every row halved."""

    def forward(self, tokens):
        return super().forward(tokens) / 2


class Adapter(torch.nn.Module):
    """A wrapper with a ``weight`` and nothing else of ``nn.Embedding``."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    @property
    def weight(self):
        return self.inner.weight

    def forward(self, tokens):
        return self.inner(tokens) + 1


def observers(m, seen):
    """Ways to see or change a call of ``m.embedding``: (name, set up, undo)."""
    note = lambda *a: seen.append(1)  # noqa: E731
    glob = torch.nn.modules.module
    e = m.embedding
    yield "forward hook", e.register_forward_hook(note)
    yield "forward pre-hook", e.register_forward_pre_hook(note)
    yield "backward hook", e.register_full_backward_hook(note)
    yield "backward pre-hook", e.register_full_backward_pre_hook(note)
    yield "global forward hook", glob.register_module_forward_hook(note)
    yield "global forward pre-hook", glob.register_module_forward_pre_hook(note)
    yield "global backward hook", glob.register_module_full_backward_hook(note)
    yield "global backward pre-hook", glob.register_module_full_backward_pre_hook(note)


DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_token_embedding_calls_what_is_more_than_a_lookup(device):
    """Subclasses, wrappers, replaced forwards and every kind of hook on the embedding
    of a TokenEmbedding are run."""
    from spikingtransformer_b200.Seq2Seq import TokenEmbedding, _only_looks_up
    tok = torch.randint(0, 9, (3, 4), generator=gen(1)).to(device)
    m = TokenEmbedding(9, 16).to(device)
    weight, scale = m.embedding.weight, 4.0
    plain = weight.detach()[tok] * scale
    assert _only_looks_up(m.embedding, tok) and torch.equal(m(tok), plain)
    seen = []
    for name, hook in observers(m, seen):
        del seen[:]
        assert not _only_looks_up(m.embedding, tok), name
        m(tok).sum().backward()
        assert seen, name
        hook.remove()
    assert _only_looks_up(m.embedding, tok)
    sub = CountedEmbedding(9, 16).to(device)
    sub.weight = weight
    m.embedding = sub
    assert torch.equal(m(tok), weight.detach()[tok] / 2 * scale)
    m.embedding = Adapter(sub)
    assert torch.equal(m(tok), (weight.detach()[tok] / 2 + 1) * scale)
    m.embedding = torch.nn.Embedding(9, 16).to(device)
    m.embedding.forward = lambda t: weight[t] * 3
    assert torch.equal(m(tok), weight.detach()[tok] * 3 * scale)
    for change in (dict(max_norm=1.0), dict(sparse=True), dict(scale_grad_by_freq=True)):
        assert not _only_looks_up(torch.nn.Embedding(9, 16, **change), tok)
    e = torch.nn.Embedding(9, 16, padding_idx=2)
    assert _only_looks_up(e, tok)
    e.padding_idx = -1  # torch counts from the end
    assert not _only_looks_up(e, tok)


@pytest.mark.parametrize("device", DEVICES)
def test_token_embedding_under_forward_mode_and_function_transforms(device):
    """Tangents, ``torch.func`` and tracing pass through a TokenEmbedding (it is linear in
    its weight: small integers, equality)."""
    import torch.autograd.forward_ad as fwd
    from torch.func import functional_call, grad, jvp, vmap
    from spikingtransformer_b200.Seq2Seq import TokenEmbedding
    m = TokenEmbedding(9, 16).to(device)
    tok = torch.randint(0, 9, (3, 4), generator=gen(1)).to(device)
    w, v = (torch.randint(-4, 5, (9, 16), generator=gen(i)).float().to(device) for i in (2, 3))
    name = "embedding.weight"

    def f(weight):
        return functional_call(m, {name: weight}, (tok,))

    out, tangent = jvp(f, (w,), (v,))
    assert torch.equal(out, w[tok] * 4) and torch.equal(tangent, v[tok] * 4)
    with fwd.dual_level():
        for leaf in (w, w.clone().requires_grad_(True)):
            assert torch.equal(fwd.unpack_dual(f(fwd.make_dual(leaf, v))).tangent, v[tok] * 4)
    counts = torch.bincount(tok.flatten(), minlength=9).float().unsqueeze(1).expand(9, 16)
    assert torch.equal(grad(lambda p: f(p).sum())(w), counts * 4)
    both = vmap(f)(torch.stack([w, v]))
    assert torch.equal(both, torch.stack([w[tok], v[tok]]) * 4)
    traced = torch.jit.trace(m, (tok,), check_trace=False)
    other = (tok + 1) % 9
    assert torch.equal(traced(other), m(other))
    compiled = torch.compile(m, backend="eager", fullgraph=True)
    assert torch.equal(compiled(other), m(other))


def test_token_embedding_is_copied_and_saved_without_its_flag():
    import copy
    import io
    from spikingtransformer_b200.Seq2Seq import TokenEmbedding
    m = TokenEmbedding(9, 16)
    tok = torch.arange(9)
    file = io.BytesIO()
    torch.save(m, file)
    file.seek(0)
    for other in (copy.deepcopy(m), copy.copy(m), torch.load(file, weights_only=False)):
        assert torch.equal(other(tok), m(tok)) and other.bad_tokens == 0
    assert copy.deepcopy(m)._watch is not m._watch
    state = dict(m.__dict__, bad_tokens=torch.ones(1))  # saved when the flag was a tensor
    del state["_watch"]
    old = TokenEmbedding.__new__(TokenEmbedding)
    old.__setstate__(state)
    assert torch.equal(old(tok), m(tok)) and old.bad_tokens == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 4096, 20000])  # tokens looked through by one block, or marked by those that meet them
@pytest.mark.parametrize("train", [False, True])
def test_token_embedding_raises_after_tokens_outside_the_vocabulary(ops, n, train):
    import copy
    from spikingtransformer_b200.Seq2Seq import TokenEmbedding
    m, other = TokenEmbedding(50, 96).to(DEV).requires_grad_(train), TokenEmbedding(60, 96).to(DEV)
    tok = torch.randint(0, 50, (n,), generator=gen(n)).to(DEV)
    want = (m.embedding.weight[tok] * 96 ** 0.5).detach()
    for wrong in (50, -1):
        bad = tok.clone()
        bad[n - 1] = wrong
        m(tok)
        m(bad)
        if wrong == 50:
            other(bad)  # inside this one's vocabulary
        torch.cuda.synchronize()
        twin = copy.deepcopy(m)
        with pytest.raises(IndexError):
            m(tok)
        for e in (m, other, twin):  # told once, and to its owner alone
            assert e.bad_tokens == 0
            e(tok)
        assert torch.equal(m(tok), want)
    m(bad)
    try:  # a later call that comes too early to see it does not clear it
        m(tok)
    except IndexError:
        return
    assert m.bad_tokens == 1


@pytest.mark.gpu
def test_token_embedding_tells_of_tokens_in_a_replayed_graph(ops):
    from spikingtransformer_b200.Seq2Seq import TokenEmbedding
    m = TokenEmbedding(50, 96).to(DEV)
    tok = torch.zeros(64, dtype=torch.int64, device=DEV)
    TokenEmbedding(2, 8).to(DEV)(tok)  # the library is loaded; m's first call is the captured one
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m(tok)
        (gw,) = torch.autograd.grad(out, m.embedding.weight, torch.ones_like(out))
    graph.replay()
    assert m.bad_tokens == 0 and torch.equal(gw[0], torch.full((96,), 64 * 96 ** 0.5, device=DEV))
    tok[5] = 77
    graph.replay()
    assert m.bad_tokens == 1
    with pytest.raises(IndexError):
        m(tok)


@pytest.mark.gpu
def test_score_is_the_log_softmax_of_the_mean_logits(ops):
    model = small_model().eval()
    g = gen(2)
    src = (torch.rand(3, 1, 32, 128, generator=g) * 0.2).to(DEV)
    tgt = torch.randint(1, 64, (3, 9), generator=g).to(DEV)
    targets = torch.randint(1, 64, (3, 9), generator=g)
    targets[1, 4:] = 0
    mask = model.create_decoder_mask(tgt, 0, DEV)
    with torch.no_grad():
        logits, _ = model(src, tgt, mask)
        logp, H, top, idx, bad = model.score(src, tgt, targets.to(DEV), mask, top_k=4, ignore_index=0)
    o = lp_exact(logits.cpu(), targets, 4, ignore=0)
    assert int(bad) == 0 and torch.equal(idx.cpu(), o["top_idx"])
    assert_within(logp, o["logp"], o["e_logp"], "logp")
    assert_within(H, o["entropy"], o["e_H"], "entropy")
    model.train()
    loss = -model.score(src, tgt, targets.to(DEV), mask, ignore_index=0)[0].sum()
    loss.backward()
    for name in ("output_layer.weight", "tgt_tok_emb.embedding.weight"):
        grad = dict(model.named_parameters())[name].grad
        assert grad is not None and torch.isfinite(grad).all() and grad.any(), name


@pytest.mark.gpu
def test_greedy_decoding_returns_its_tokens_log_probabilities(ops):
    model = small_model().eval()
    src = (torch.rand(4, 1, 32, 128, generator=gen(5)) * 0.2).to(DEV)
    ys, lengths = model.greedy_decode_batch(src, 8, 1, 2, 0)
    ys2, lengths2, logp = model.greedy_decode_batch(src, 8, 1, 2, 0, return_logprobs=True)
    assert torch.equal(ys, ys2) and torch.equal(lengths, lengths2) and logp.shape == ys.shape
    assert not logp[:, 0].any()
    for b in range(4):
        n = int(lengths[b])
        assert not logp[b, n:].any()
        # the last token again, from the whole prefix before it
        pre = ys[b:b + 1, :n - 1]
        with torch.no_grad():
            enc, _ = model.encode(src[b:b + 1])
            out, _ = model.decode(pre, enc, model.create_decoder_mask(pre, 0, DEV))
        o = lp_exact(out[:, :, -1].cpu(), ys[b, n - 1:n].cpu(), 0)
        assert_within(logp[b, n - 1:n], o["logp"], o["e_logp"] + 1e-5, "logp")


# ------------------------------------------------------------------ together, streams, graphs


def chain(ops, tok, tgt, w, gamma, beta, out_w):
    h, _ = ops.embedding(tok, w, w.shape[1] ** 0.5)
    y = ops.layer_norm(h, gamma, beta)
    return ops.token_logprobs((y @ out_w.t()).unsqueeze(0), tgt, top_k=3)


def chain_inputs(seed, V=300, D=96, B=4, N=33):
    g = gen(seed)
    tok = torch.randint(0, V, (B, N), generator=g).to(DEV)
    tgt = torch.randint(0, V, (B, N), generator=g).to(DEV)
    ps = [torch.randn(V, D, generator=g) * 0.1, 1 + 0.1 * torch.randn(D, generator=g),
          0.1 * torch.randn(D, generator=g), torch.randn(V, D, generator=g) * 0.1]
    return tok, tgt, [p.to(DEV).requires_grad_(True) for p in ps]


@pytest.mark.gpu
def test_the_operators_together_train_as_the_plain_model(ops):
    """Embedding, LayerNorm, projection and log probabilities in a row, fp32, against
    the same in 64 bits: errors of about 1e-6 a stage of values of order 1."""
    tok, tgt, ps = chain_inputs(1)
    logp, H, top, idx, _ = chain(ops, tok, tgt, *ps)
    loss = -logp.mean() - 0.01 * H.mean() + 0.1 * top.mean()
    grads = torch.autograd.grad(loss, ps)
    qs = [p.detach().double().requires_grad_(True) for p in ps]
    w, gamma, beta, out_w = qs
    h = w[tok] * w.shape[1] ** 0.5
    y = torch.nn.functional.layer_norm(h, (h.shape[-1],), gamma, beta)
    lp = (y @ out_w.t()).log_softmax(-1)
    H2 = -(lp.exp() * lp).sum(-1)
    loss = loss.detach()
    loss2 = -lp.gather(-1, tgt[..., None]).mean() - 0.01 * H2.mean() + 0.1 * lp.gather(-1, idx).mean()
    assert abs(float(loss) - float(loss2.detach())) < 1e-5
    for a, b in zip(grads, torch.autograd.grad(loss2, qs)):
        # K = 96 and 132-row fp32 products (at most 132 u of the terms' size) dominate
        assert (a.double() - b).abs().max() <= 2e-5 * b.abs().max()


@pytest.mark.gpu
def test_operators_on_another_stream(ops):
    tok, tgt, ps = chain_inputs(2)
    want = chain(ops, tok, tgt, *ps)
    gw = torch.autograd.grad(want[0].sum(), ps)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain(ops, tok, tgt, *ps)
        gg = torch.autograd.grad(got[0].sum(), ps)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(list(want) + list(gw), list(got) + list(gg)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_operators_in_two_cuda_graphs(ops):
    """Forward and backward captured twice (each graph with buffers of its own),
    replayed in turn on new inputs: the eager results."""
    def static(seed):
        tok, tgt, ps = chain_inputs(seed)
        return tok, tgt, ps

    def step(s):
        out = chain(ops, s[0], s[1], *s[2])
        return list(out) + list(torch.autograd.grad(out[0].sum() + out[1].sum(), s[2]))

    made = []
    for seed in (3, 4):
        s = static(seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(s)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(s)
        made.append((s, graph, outs))
    for seed in (5, 6):
        for s, graph, _ in made:
            new = static(seed)
            s[0].copy_(new[0])
            s[1].copy_(new[1])
            with torch.no_grad():
                for p, q in zip(s[2], new[2]):
                    p.copy_(q)
            graph.replay()
    torch.cuda.synchronize()
    for s, graph, outs in made:
        for a, b in zip(outs, step(s)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(ops):
    """Tensors of more than 2^31 elements: the last rows equal those of a small call."""
    D, rows = 2048, (1 << 20) + 4096
    x = torch.empty(rows, D, dtype=torch.bfloat16, device=DEV).normal_()
    w = torch.randn(D, device=DEV)
    y, stats = ops.layer_norm_fwd(x, w)
    assert torch.equal(y[-64:], ops.layer_norm(x[-64:], w))
    gx, _, _ = ops.layer_norm_bwd(x, x, stats, w, need_weight=False, need_bias=False)
    assert torch.equal(gx[-64:], ops.layer_norm_bwd(x[-64:], x[-64:], stats[-64:], w)[0])
    del y, gx
    tok = torch.tensor([0, rows - 1, rows - 1, 1 << 20, 7], device=DEV)
    out, bad = ops.embedding(tok, x)
    assert int(bad) == 0 and torch.equal(out, x[tok])
    g = torch.randint(-9, 10, (5, D), device=DEV).to(torch.bfloat16)
    gw = ops.embedding_bwd(g, tok, rows, dtype=torch.bfloat16)
    assert torch.equal(gw[rows - 1], g[1] + g[2]) and torch.equal(gw[0], g[0]) and torch.equal(gw[1 << 20], g[3])
    assert not gw[rows - 2].any() and float(gw[-4000:].float().abs().sum()) == float((g[1] + g[2]).float().abs().sum())
    del gw
    big = torch.randint(0, rows, (rows,), device=DEV)
    out, _ = ops.embedding(big, x[:, :D])
    assert torch.equal(out[-1000:], x[big[-1000:]])
    del out, big
    V = 65536
    z = x.flatten()[: (1 << 15) * V + 64 * V].view(1, -1, V)
    t = torch.randint(0, V, (z.shape[1],), device=DEV)
    logp, H, top, idx, _ = ops.token_logprobs(z, t, top_k=2)
    last = ops.token_logprobs(z[:, -64:], t[-64:], top_k=2)
    # 64 rows are cut over several blocks and join their sums in another order
    for a, b in zip((logp, H, top), last):
        assert torch.allclose(a[-64:], b, rtol=0, atol=2e-5)
    assert torch.equal(idx[-64:], last[3])
    zl = z.detach().requires_grad_(True)
    (gz,) = torch.autograd.grad(ops.token_logprobs(zl, t)[0].sum(), zl)
    p = z[0, -1].float().softmax(-1)
    p[t[-1]] -= 1.0
    assert torch.allclose(gz[0, -1].float(), -p, rtol=2 ** -7, atol=1e-8)


@pytest.mark.gpu
def test_operators_run_beside_each_other(ops):
    """The same calls at once on two streams, each with its own buffers."""
    a, b = chain_inputs(21), chain_inputs(22)
    want = [torch.autograd.grad(chain(ops, s[0], s[1], *s[2])[0].sum(), s[2]) for s in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                ps = [p.detach().requires_grad_(True) for p in s[2]]
                got[i].append(torch.autograd.grad(chain(ops, s[0], s[1], *ps)[0].sum(), ps))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        for r in runs:
            assert all(torch.equal(u, v) for u, v in zip(w, r))


@pytest.mark.gpu
def test_operators_from_several_threads(ops):
    """Calls of different sizes (and so of different shared memory) from four host
    threads at once give what they give one after the other."""
    import threading
    sizes = [(64, 512, torch.float32), (300, 768, torch.float32), (33, 8192, torch.float32), (50, 96, torch.bfloat16)]

    def work(rows, D, dtype, seed):
        x, w, b, gy = (t.to(DEV) for t in ln_case(rows, D, dtype, seed))
        res = []
        for _ in range(20):
            y, stats = ops.layer_norm_fwd(x, w, b)
            res = [y, *ops.layer_norm_bwd(gy, x, stats, w)]
            tok = torch.arange(rows, device=DEV) * 7919 % (1 << (8 + seed))
            res.append(ops.embedding_bwd(gy, tok, 1 << (8 + seed)))
            res += ops.token_logprobs(x[None], tok % D, top_k=min(seed + 1, D))[:4]
        torch.cuda.current_stream().synchronize()
        return res

    want = [work(*s, i) for i, s in enumerate(sizes)]
    got, errors = [None] * len(sizes), []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got[i] = work(*sizes[i], i)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(sizes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.gpu
def test_no_device_timeouts(ops):
    ops.device_error_check()
