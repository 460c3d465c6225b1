"""Values of a trainer's operators (p2pdl_amd/training.py) at the ends of their types' ranges, and what a
call may not depend on: where its operands lie, which host path made it.

Bounds as in test_training_ops.py, whose forms in 64 bits these tests share; `strict` compares infinities
and NaN too.
"""
import pytest
import torch

import test_training_ops as ops
from p2pdl_amd import _native as N
from p2pdl_amd import training as T
from test_training_ops import DTYPES, U, gpu, randn, rounded, same_bits


def strict(got, want, bound, what):
    """|got - want| <= bound wherever want is finite, the same infinity or a NaN elsewhere."""
    got, want, bound = got.detach().double().cpu(), want.double().cpu(), bound.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), (what, "NaN")
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)]), (what, "infinities")
    fine = torch.isfinite(want)
    assert torch.isfinite(bound.expand_as(want)[fine]).all(), (what, "no bound")
    bad = fine & ~((got - want).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((got - want).abs()[bad].max()))


# ------------------------------------------------------------------ layer norm
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [1, 3, 8, 10, 24, 100])
def test_layer_norm_backward_of_large_constant_rows(cuda, dtype, cols):
    """A constant row of 2^120: rstd is 1 / sqrt(eps), so (0 - mean) * rstd leaves float32's range in the lanes past
    the row, which add nothing.  Its sums are exact, x - mean is 0: dx = rstd * (g - mean(g)) and dw = 0."""
    x = torch.full((5, cols), 2.0 ** 120, dtype=dtype, device="cuda")
    x[1::2] = 0.5
    dy, w = randn((5, cols), dtype, 70), randn((cols,), dtype, 71)
    y, mean, rstd = T.layer_norm_forward(x, w)
    assert torch.equal(mean, x[:, 0].float()) and not y.any()
    dx, dw, db = T.layer_norm_backward(dy, x, mean, rstd, w)
    g, r = dy.double().cpu() * w.double().cpu(), rstd.double().cpu()[:, None]
    want = r * (g - g.mean(1, keepdim=True))
    bound = r * 16 * U * (g.abs() + g.abs().mean(1, keepdim=True))
    strict(dx, want, rounded(want, bound, dtype), "dx")
    strict(dw, torch.zeros(cols), torch.zeros(cols), "dw")
    total = dy.double().cpu().sum(0)
    strict(db, total, rounded(total, 16 * U * dy.double().cpu().abs().sum(0), dtype), "db")


# ------------------------------------------------------------------ gated linear layer
GATED_RANGE = [(30, 64, 40), (600, 264, 500), (257, 2041, 1100), (1500, 512, 300)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,units", GATED_RANGE)
@pytest.mark.parametrize("grad,up", [(2.0 ** -22, 1.0), (2.0 ** -22, 64.0), (2.0 ** -17, 1.0), (100.0, 300.0)])
def test_gated_linear_small_and_large_gradients(cuda, monkeypatch, dtype, rows, cols, units, grad, up):
    """dg and du next to either end of float16's range, on the small path and on tiles: their rounding is half a step
    of the type, or of float16's smallest one scaled (the largest is held in [2^14, 2^15): 2^-25 * 2^-14 of it)."""
    x, dh = randn((rows, cols), dtype, 72), randn((rows, units), dtype, 73, grad)
    wg, wu = randn((units, cols), dtype, 74, cols ** -0.5), randn((units, cols), dtype, 75, cols ** -0.5 * up)
    h, gate, u_ = T.gated_linear_forward(x, wg, wu)
    got = T.gated_linear_backward(dh, x, wg, wu, gate, u_)
    a, da = ops.act64("silu", x.double().cpu() @ wg.double().cpu().t())
    d64 = dh.double().cpu()
    largest = max((d64 * da * (x.double().cpu() @ wu.double().cpu().t())).abs().max(), (d64 * a).abs().max()).item()

    def scaled(want, err, t):
        floor = 2.0 ** -39 * 1.01 * largest if t == torch.float16 else ops.tiny(t)
        return err + ops.u(t) * (want.abs() + err) + floor

    with monkeypatch.context() as m:
        m.setattr(ops, "rounded", scaled)  # of dg and du; the results' own roundings are the type's
        want, err = ops.gated_reference(x, wg, wu, dh, "silu")
    for o, v, e, name in zip(got, want[1:], err[1:], ("dx", "dwg", "dwu")):
        bound = rounded(v, e, dtype)
        # rounded to the type: what is past its largest value is an infinity; at that border either may come
        limit = torch.finfo(dtype).max
        clear = ((v.abs() + bound) < limit) | ((v.abs() - bound) > limit * (1 + ops.u(dtype)))
        v = torch.where(v.abs() > limit, torch.copysign(torch.tensor(float("inf"), dtype=v.dtype), v), v)
        strict(torch.where(clear, o.double().cpu(), 0.0), torch.where(clear, v, 0.0), bound, (name, largest))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,units", GATED_RANGE[:2])
def test_gated_linear_gradients_that_are_not_finite(cuda, dtype, rows, cols, units):
    """A NaN and an infinity in one token's dh stay with that token's dx; the other tokens' dx have the bits they have
    without them (the power of two of float16 goes by the finite ones)."""
    x, dh = randn((rows, cols), dtype, 76), randn((rows, units), dtype, 77)
    wg, wu = randn((units, cols), dtype, 78, cols ** -0.5), randn((units, cols), dtype, 79, cols ** -0.5)
    h, gate, up = T.gated_linear_forward(x, wg, wu)
    clean = T.gated_linear_backward(dh, x, wg, wu, gate, up)[0]
    bad = dh.clone()
    bad[3, 5], bad[7, 9] = float("nan"), float("inf")
    dx, dwg, dwu = T.gated_linear_backward(bad, x, wg, wu, gate, up)
    rest = [i for i in range(rows) if i not in (3, 7)]
    assert same_bits(dx[rest], clean[rest]) and not torch.isfinite(dx[[3, 7]]).any()
    assert not torch.isfinite(dwg[[5, 9]]).any() and not torch.isfinite(dwu[[5, 9]]).any()
    others = [i for i in range(units) if i not in (5, 9)]
    assert torch.isfinite(dwg[others]).all() and torch.isfinite(dwu[others]).all()
    # nothing to scale by: no gradient, and none that is finite
    zero = T.gated_linear_backward(torch.zeros_like(dh), x, wg, wu, gate, up)
    assert not any(t.any() for t in zero)
    assert torch.isnan(T.gated_linear_backward(torch.full_like(dh, float("nan")), x, wg, wu, gate, up)[0]).all()


@gpu
def test_captured_float16_gradients_are_scaled_by_their_own(cuda):
    """A captured backward pass finds the power of two of the values that it is replayed on: gradients 2^30 apart, an
    infinity, zeros and the first ones again, with eager passes of other sizes between the replays."""
    rows, cols, units = 600, 264, 500
    x, base = randn((rows, cols), torch.float16, 93), randn((rows, units), torch.float16, 94)
    wg, wu = (randn((units, cols), torch.float16, s, cols ** -0.5) for s in (95, 96))
    h, gate, up = T.gated_linear_forward(x, wg, wu)
    dh = base.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        T.gated_linear_backward(dh, x, wg, wu, gate, up)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = T.gated_linear_backward(dh, x, wg, wu, gate, up)
    for factor in (1.0, 2.0 ** -18, 4096.0, float("inf"), 0.0, 1.0):
        dh.copy_(base)
        if factor != float("inf"):
            dh.mul_(factor)
        else:
            dh[3, 5] = factor
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        T.gated_linear_backward(base[:300], x[:300], wg, wu, gate[:300], up[:300])
        want = T.gated_linear_backward(dh, x, wg, wu, gate, up)
        assert all(same_bits(a, b) for a, b in zip(got, want)), factor


# ------------------------------------------------------------------ linear cross entropy
@pytest.mark.parametrize("dtype", [N.P2P_DTYPE_F16, N.P2P_DTYPE_BF16])
@pytest.mark.parametrize("tokens,hidden,vocab", [(256, 4096, 70000), (1024, 4096, 131072), (2048, 4096, 131072), (512, 2048, 400000)])
@pytest.mark.parametrize("backward", [0, 1])
def test_linear_ce_pieces_do_not_depend_on_the_weights_place(dtype, tokens, hidden, vocab, backward):
    """A weight that cannot be read where it lies costs its copy; the pieces, whose sums are rounded one by one, stay."""
    L = N.load_library()
    here = ops.ce_args(tokens=tokens, hidden=hidden, vocab=vocab, ldx=hidden, ldw=hidden, dtype=dtype)
    need = L.p2p_linear_ce_workspace(here, backward)
    for other in ({"w": here.w + 2}, {"ldw": hidden + 1}):
        there = ops.ce_args(tokens=tokens, hidden=hidden, vocab=vocab, ldx=hidden, ldw=hidden, dtype=dtype)
        for k, v in other.items():
            setattr(there, k, v)
        assert L.p2p_linear_ce_workspace(there, backward) - need == vocab * hidden * 2, other


@gpu
def test_linear_cross_entropy_bits_do_not_depend_on_the_weights_place(cuda):
    """256 x 4096 x 70000: the copy of a weight that lies one element off, or has an odd pitch, is 573 MB."""
    rows, cols, vocab = 256, 4096, 70000
    g = torch.Generator("cuda").manual_seed(80)
    w = torch.randn((vocab, cols), generator=g, device="cuda", dtype=torch.bfloat16) * 0.03
    x = torch.randn((rows, cols), generator=g, device="cuda", dtype=torch.bfloat16)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    dloss = torch.tensor(256.0, device="cuda")

    def step(weight):
        loss, lse, norm = T.linear_cross_entropy_forward(x, weight, t)
        return (loss, lse) + T.linear_cross_entropy_backward(x, weight, t, lse, norm, dloss)

    want = step(w)
    off = torch.empty(vocab * cols + 1, device="cuda", dtype=w.dtype)[1:].view(vocab, cols).copy_(w)
    pitched = torch.empty((vocab, cols + 1), device="cuda", dtype=w.dtype)[:, :cols].copy_(w)
    for other in (off, pitched):
        assert all(same_bits(a, b) for a, b in zip(step(other), want))


# ------------------------------------------------------------------ both host paths
def host_paths(monkeypatch):
    """'C++', then 'Python': the path that a dense call takes, and the one that copies and explains."""
    yield "C++"
    with monkeypatch.context() as m:
        m.setattr(T, "_host", type("NoHost", (), {"__getattr__": lambda self, name: lambda *a: None})())
        yield "Python"


@gpu
@pytest.mark.parametrize("pitched", [False, True])
def test_a_loss_may_be_changed_in_place(cuda, monkeypatch, pitched):
    """loss /= steps before backward(), whichever path made the loss."""
    wide = randn((12, 40), torch.float32, 81)
    x = wide[:, 3:35] if pitched else wide[:, :32].contiguous()
    t = (torch.arange(12) % 7).cuda()
    grads = []
    for path in host_paths(monkeypatch):
        w = randn((7, 32), torch.float32, 82).requires_grad_()
        loss = T.linear_cross_entropy(x, w, t)
        loss /= 4
        loss.mul_(2)
        loss.backward()
        grads.append(w.grad)
    assert same_bits(*grads)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_results_are_tensors_of_their_own(cuda, monkeypatch, dtype):
    """No result is a view, or shares its memory with another one, and both paths have the same bits."""
    x, dy = randn((9, 24), dtype, 83), randn((9, 24), dtype, 84)
    w, wide, dh = randn((24,), dtype, 85), randn((16, 24), dtype, 86), randn((9, 16), dtype, 87)
    t = (torch.arange(9) % 16).cuda()
    found = []
    for path in host_paths(monkeypatch):
        y, mean, rstd = T.layer_norm_forward(x, w, w)
        h, gate, up = T.gated_linear_forward(x, wide, wide)
        loss, lse, norm = T.linear_cross_entropy_forward(x, wide, t)
        out = [y, mean, rstd, h, gate, up, loss, lse, norm, T.dropout_forward(x, 0.5, 3, residual=x)]
        out += T.layer_norm_backward(dy, x, mean, rstd, w)
        out += T.gated_linear_backward(dh, x, wide, wide, gate, up)
        out += T.linear_cross_entropy_backward(x, wide, t, lse, norm)
        out += T.layer_norm_backward(dy[:0], x[:0], mean[:0], rstd[:0], w)[1:]
        assert all(o._base is None for o in out), path
        assert len({o.untyped_storage().data_ptr() for o in out}) == len(out), path
        found.append(out)
    assert all(same_bits(a, b) for a, b in zip(*found))
    assert not found[0][-1].any() and not found[0][-2].any()


# ------------------------------------------------------------------ limits
def test_limits_are_the_librarys():
    """The wrappers' limits are the library's own, on either side of each."""
    L = N.load_library()
    n, f = T.MAX_UNITS, T.MAX_FEATURES
    assert L.p2p_gated_linear_workspace(ops.gated_args(units=n), 1) >= 0
    assert L.p2p_gated_linear_workspace(ops.gated_args(units=n + 1), 1) == -2
    wide = {"hidden": f, "ldx": f, "ldg": f, "ldu": f}
    assert L.p2p_gated_linear_workspace(ops.gated_args(**wide), 1) >= 0
    assert L.p2p_gated_linear_workspace(ops.gated_args(**{k: v + 1 for k, v in wide.items()}), 1) == -2
    wide = {"hidden": f, "ldx": f, "ldw": f}
    assert L.p2p_linear_ce_workspace(ops.ce_args(**wide), 1) >= 0
    assert L.p2p_linear_ce_workspace(ops.ce_args(**{k: v + 1 for k, v in wide.items()}), 1) == -2
    c = T.MAX_NORM_COLS
    assert L.p2p_layernorm_bwd_workspace(1, c, 0) >= 0 and L.p2p_layernorm_bwd_workspace(1, c + 1, 0) < 0


@gpu
def test_more_units_than_the_limit_are_refused(cuda):
    """2^21 - 8 units run; past them, up to 2^21 - 4 and more, both passes say what the limit is."""
    x = torch.ones(1, 1, device="cuda")
    for n in (T.MAX_UNITS, T.MAX_UNITS + 1, T.MAX_UNITS + 4, T.MAX_UNITS + 5):
        w = torch.ones(n, 1, device="cuda")
        row = torch.ones(1, n, device="cuda")
        if n == T.MAX_UNITS:
            h, gate, up = T.gated_linear_forward(x, w, w, "relu")
            assert (h == 1).all() and T.gated_linear_backward(row, x, w, w, gate, up, "relu")[0].item() == 2 * n
            continue
        for call in (lambda: T.gated_linear_forward(x, w, w, "relu"),
                     lambda: T.gated_linear_backward(row, x, w, w, row, row, "relu")):
            with pytest.raises(ValueError, match=str(T.MAX_UNITS)):
                call()


# ------------------------------------------------------------------ the forms in 64 bits, infinities and NaN compared too
def reruns():
    for dtype in DTYPES:
        for shape in ops.NORM_SHAPES:
            yield ops.test_layer_norm, (dtype, *shape)
        for shape in ops.GATED_SHAPES:
            yield ops.test_gated_linear, (dtype, *shape, "silu")
        for shape in ops.CE_SHAPES:
            yield ops.test_linear_cross_entropy, (dtype, *shape, "mean")
        for args in ((1000, 0.1, 0xDEADBEEFCAFEF00D, (1 << 32) - 3), (2051, 1 - 2.0 ** -33, 3, 4)):
            yield ops.test_dropout, (dtype, *args)


@gpu
@pytest.mark.parametrize("test,args", [pytest.param(t, a, id=f"{t.__name__[5:]}-{'-'.join(str(v) for v in a)}") for t, a in reruns()])
def test_values_that_are_not_finite_too(cuda, monkeypatch, test, args):
    """ops.check lets a value pass where the form in 64 bits has a NaN or an infinity; here none does."""
    monkeypatch.setattr(ops, "check", strict)
    test(cuda, *args)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,units", [(30, 64, 40), (600, 264, 500)])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gated_linear_inputs_that_are_not_finite(cuda, dtype, rows, cols, units, act):
    """A NaN and an infinity in x: what the form in 64 bits makes of them, in every place.  (An infinity among
    the float32 operands of a product on tiles may come out as NaN.)"""
    x, dh = randn((rows, cols), dtype, 88), randn((rows, units), dtype, 89)
    wg, wu = randn((units, cols), dtype, 90, cols ** -0.5), randn((units, cols), dtype, 91, cols ** -0.5)
    x[3, 5] = float("nan")
    if dtype != torch.float32 or rows <= 192:
        x[7, 9] = float("inf")
    h, gate, up = T.gated_linear_forward(x, wg, wu, act)
    got = (h,) + T.gated_linear_backward(dh, x, wg, wu, gate, up, act)
    want, err = ops.gated_reference(x, wg, wu, dh, act)
    for o, v, e, name in zip(got, want, err, ("h", "dx", "dwg", "dwu")):
        strict(o, v, rounded(v, e, dtype), name)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,vocab", [(30, 64, 100), (600, 264, 900)])
def test_linear_cross_entropy_inputs_that_are_not_finite(cuda, dtype, rows, cols, vocab):
    """A NaN in a token that counts: the loss, that token's dx and all of dW; no other token's dx."""
    x, w, t = ops.ce_inputs(rows, cols, vocab, dtype, 92)
    t[3] = 5
    loss, lse, norm = T.linear_cross_entropy_forward(x, w, t)
    clean = T.linear_cross_entropy_backward(x, w, t, lse, norm)[0]
    x[3, 6] = float("nan")
    loss, lse, norm = T.linear_cross_entropy_forward(x, w, t)
    dx, dw = T.linear_cross_entropy_backward(x, w, t, lse, norm)
    rest = [i for i in range(rows) if i != 3]
    assert torch.isnan(loss) and torch.isnan(lse[3]) and torch.isfinite(lse[rest]).all()
    assert torch.isnan(dx[3]).all() and same_bits(dx[rest], clean[rest]) and torch.isnan(dw).all()


@gpu
def test_an_error_inside_a_call_is_the_callers(cuda):
    """What `save` raises when it is asked for its truth comes out as it is, and the next call is as before."""
    x, w = torch.ones(2, 8, device="cuda"), torch.ones(4, 8, device="cuda")
    want = T.gated_linear_forward(x, w, w)
    with pytest.raises(RuntimeError, match="[Bb]oolean"):
        T.gated_linear_forward(x, w, w, save=torch.ones(2))
    assert all(same_bits(a, b) for a, b in zip(T.gated_linear_forward(x, w, w, save=torch.ones(())), want))
