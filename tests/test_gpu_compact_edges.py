"""Compact-scene operators on the MI355X: calls at the edges of autograd, of their arguments and of the launch rules
(tests/test_gpu_compact.py has the values)."""
import pytest
import torch

from test_gpu_compact import DEV, both_routes, gen, model, scene

pytestmark = pytest.mark.gpu


def test_evict_of_groups_that_can_be_read_once():
    """Groups from an iterator (zip(begins, ends)): the same Gaussians as from a list."""
    a, b = model(), model()
    budgets = [500, 900]
    want, ranges = a.evict(budgets, recent=[100, 0], groups=[(0, 1000), (1000, 3000)])
    got, again = b.evict(budgets, recent=[100, 0], groups=zip([0, 1000], [1000, 3000]))
    assert again == ranges == [(0, 500), (500, 1400)] and b.num_points == 1400
    assert torch.equal(got, want) and torch.equal(a._arena.data, b._arena.data)
    c, d = model(), model()
    want, ranges = c.evict(700, groups=[(0, 1000), (1000, 3000)])
    got, again = d.evict(700, groups=iter([(0, 1000), (1000, 3000)]))  # one budget for all of them
    assert again == ranges and d.num_points == 1400 and torch.equal(got, want)


def test_evict_with_weights_of_another_number():
    m = model()
    m.contribution = torch.zeros(2999, 1, device=DEV)
    with pytest.raises(RuntimeError, match="contribution must hold 3000"):
        m.evict(100)
    assert m.num_points == 3000


# ---- derivatives that there are none of -----------------------------------------------------------
def test_second_derivatives_are_refused_under_a_linear_loss(monkeypatch):
    """The first gradients depend on the inputs even where the upstream gradient is a constant: dxyz on xyz and on
    the coefficients, dfeatures on xyz.  All of these are refused, by backward() and by grad() of one input."""
    import gsr_train as G
    xyz, f, cam, up = scene(40, 16, 2, 3)
    xyz, f, cam, up = (t.to(DEV) for t in (xyz, f, cam, up))
    rest = G.mx4_quantize(f.flatten(1)[:, 3:])

    def fresh():
        return [t.clone().requires_grad_() for t in (xyz, f, f[:, 0])]

    def refused(run):
        with pytest.raises(RuntimeError, match="once_differentiable"):
            run()

    for _ in both_routes(monkeypatch):
        x, fg, dc = fresh()
        first = lambda c, *of: torch.autograd.grad((c * up).sum(), of, create_graph=True)  # noqa: E731
        trained = lambda: G.sh_colors_quantized(x, fg, cam, 3)  # noqa: E731
        shown = lambda: G.sh_colors(x, dc, rest, cam, 3)  # noqa: E731
        (gx,) = first(trained(), x)
        refused(lambda: (gx.square().sum() + x.sum()).backward())
        (gx,) = first(trained(), x)
        refused(lambda: torch.autograd.grad(gx.square().sum() + x.sum(), x))
        (gx,) = first(trained(), x)
        refused(lambda: torch.autograd.grad(gx.sum() + fg.sum(), fg))
        gx, gf = first(trained(), x, fg)
        refused(lambda: torch.autograd.grad(gf.square().sum() + x.sum(), x))
        (gx,) = first(shown(), x)
        refused(lambda: (gx.square().sum() + x.sum()).backward())
        (gx,) = first(shown(), x)
        refused(lambda: torch.autograd.grad(gx.sum() + x.sum(), x))
        # an upstream gradient that is a function of something
        gd, = torch.autograd.grad(shown().square().sum(), dc, create_graph=True)
        refused(lambda: torch.autograd.grad(gd.sum() + dc.sum(), dc))


def test_first_gradients_that_are_constants_stay_usable(monkeypatch):
    """What a second derivative would be zero of: the constants' gradient under a constant upstream gradient, the
    features' one when the positions are fixed, everything at degree 0."""
    import gsr_train as G
    xyz, f, cam, up = (t.to(DEV) for t in scene(40, 16, 2, 3))
    rest = G.mx4_quantize(f.flatten(1)[:, 3:])
    for _ in both_routes(monkeypatch):
        x, fg, dc = [t.clone().requires_grad_() for t in (xyz, f, f[:, 0])]
        cases = [(G.sh_colors(x, dc, rest, cam, 3), dc, dc), (G.sh_colors_quantized(xyz, fg, cam, 3), fg, fg),
                 (G.sh_colors_quantized(x, fg, cam, 0), fg, fg), (G.sh_colors_quantized(x, fg, cam, 0), x, x)]
        for c, of, leaf in cases:
            (want,) = torch.autograd.grad(c, of, up, retain_graph=True)
            (g,) = torch.autograd.grad(c, of, up, create_graph=True)
            assert torch.equal(g, want)
            (one,) = torch.autograd.grad(g.square().sum() + leaf.sum(), leaf)
            assert (one == 1).all()


def test_forward_mode_is_refused(monkeypatch):
    """A tangent on an input would be lost: no colours without it."""
    import gsr_train as G
    import torch.autograd.forward_ad as fw
    xyz, f, cam, _ = (t.to(DEV) for t in scene(20, 4, 1, 8))
    rest = G.mx4_quantize(f.flatten(1)[:, 3:])
    dc = f[:, 0].contiguous()
    for _ in both_routes(monkeypatch):
        shown, trained = G.sh_colors(xyz, dc, rest, cam, 1), G.sh_colors_quantized(xyz, f, cam, 1)
        with fw.dual_level():
            dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
            for call in (lambda: G.sh_colors(dual(xyz), dc, rest, cam, 1), lambda: G.sh_colors(xyz, dual(dc), rest, cam, 1),
                         lambda: G.sh_colors(xyz, dc, rest, dual(cam), 1),
                         lambda: G.sh_colors_quantized(dual(xyz), f, cam, 1),
                         lambda: G.sh_colors_quantized(xyz, dual(f), cam, 1),
                         lambda: G.sh_colors_quantized(xyz, f, dual(cam), 1)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                    call()
            # other tensors of the level do not matter
            assert torch.equal(G.sh_colors(xyz, dc, rest, cam, 1), shown)
            assert torch.equal(G.sh_colors_quantized(xyz, f, cam, 1), trained)


# ---- tracing --------------------------------------------------------------------------------------
def test_traced_colors_are_computed(monkeypatch):
    """A traced call runs the operator on the new inputs (a recorded allocation without the kernel would be
    uninitialised memory), with gradients."""
    import gsr_train as G
    xyz, f, cam, up = (t.to(DEV) for t in scene(200, 9, 2, 14))
    other, f2, cam2, _ = (t.to(DEV) for t in scene(200, 9, 2, 15))
    rest = G.mx4_quantize(f.flatten(1)[:, 3:])
    for _ in both_routes(monkeypatch):
        for trained in (True, False):
            if trained:
                fn = lambda x, c, k: G.sh_colors_quantized(x, c, k, 2)  # noqa: E731
            else:
                fn = lambda x, c, k: G.sh_colors(x, c[:, 0], rest, k, 2)  # noqa: E731
            for grad in (False, True):
                x, c = xyz.clone().requires_grad_(grad), f.clone().requires_grad_(grad)
                traced = torch.jit.trace(fn, (x, c, cam), check_trace=False)
                x, c = other.clone().requires_grad_(grad), f2.clone().requires_grad_(grad)
                got, want = traced(x, c, cam2), fn(x, c, cam2)
                assert torch.equal(got, want)
                if grad:
                    for a, b in zip(torch.autograd.grad(got, (x, c), up), torch.autograd.grad(want, (x, c), up)):
                        assert torch.equal(a, b)


def test_other_operators_refuse_to_be_traced(monkeypatch):
    import gsr_train as G
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.randn(100, 45, generator=gen(1)).to(DEV)
    w = torch.rand(100, generator=gen(2)).to(DEV)
    ids = torch.arange(10, dtype=torch.int32, device=DEV)
    rows = G.mx4_quantize(x)
    xyz, f, cam, _ = (t.to(DEV) for t in scene(20, 4, 1, 8))
    rest = G.mx4_quantize(f.flatten(1)[:, 3:])
    calls = [(lambda t: G.mx4_quantize(t).codes, x), (lambda t: rows.dequantize() + t[:1], x),
             (lambda t: G.keep_heaviest(t, 5), w), (lambda t: G.take_rows(ids, [t])[0], x)]
    for _ in both_routes(monkeypatch):
        for fn, arg in calls:
            with pytest.raises(RuntimeError, match="traced"):
                torch.jit.trace(fn, (arg,), check_trace=False)
            with pytest.raises(RuntimeError, match="traced"):
                make_fx(fn)(arg)
        acc = torch.zeros(100, device=DEV)

        def add(t):
            G.accumulate_weights(acc, t)
            return t + 0

        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(add, (w,), check_trace=False)
        assert (acc == 0).all()
        for fn in (lambda t: G.sh_colors_quantized(t, f, cam, 1), lambda t: G.sh_colors(t, f[:, 0], rest, cam, 1)):
            with pytest.raises(RuntimeError, match="traced"):
                make_fx(fn)(xyz)


# ---- writes in place ------------------------------------------------------------------------------
def test_writes_in_place_are_seen_by_autograd(monkeypatch):
    """A tensor that another graph has saved cannot be written behind its back."""
    import gsr_train as G
    ids = torch.arange(5, dtype=torch.int32, device=DEV)
    for _ in both_routes(monkeypatch):
        x = torch.randn(5, 3, device=DEV).requires_grad_()
        acc, out = torch.rand(5, device=DEV), torch.rand(5, 3, device=DEV)
        loss = (x[:, 0] * acc).sum()
        G.accumulate_weights(acc, torch.ones(5, device=DEV))
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        loss = (x * out).sum()
        G.take_rows(ids, [torch.rand(9, 3, device=DEV)], out=[out])
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        # a refused call has written nothing
        loss = (x * out).sum()
        with pytest.raises(RuntimeError, match="overlaps"):
            G.take_rows(ids, [out], out=[out])
        loss.backward()
        # tensors without a version counter
        with torch.inference_mode():
            acc, out = torch.zeros(5, device=DEV), torch.zeros(5, 3, device=DEV)
            G.accumulate_weights(acc, torch.ones(5, device=DEV))
            G.take_rows(ids, [torch.ones(9, 3, device=DEV)], out=[out])
        assert (acc == 1).all() and (out == 1).all()


def test_weights_beside_and_between_their_sums():
    """acc in the middle of the memory that the weights are a strided view of: allowed where they share no element or
    none but an element's own, each result that of separate tensors."""
    import gsr_train as G
    for P, start, stride in ((10, 50, 1), (1, 50, 5), (10, 60, 1), (10, 40, 1), (10, 49, 11), (10, 49, 0), (10, 60, 0),
                             (5, 48, 30), (10, 10, 4), (4, 44, 10),
                             (7, 30, 6)):
        buf = torch.rand(400, generator=gen(P * stride + start)).to(DEV)
        acc, w = buf[50:50 + P], buf.as_strided((P,), (stride,), start)
        want = acc.clone()
        G.accumulate_weights(want, w.clone(), 0.5)
        before = buf.clone()
        G.accumulate_weights(acc, w, 0.5)
        assert torch.equal(acc, want), (P, start, stride)
        before[50:50 + P] = want
        assert torch.equal(buf, before)
    for P, start, stride in ((10, 51, 1), (10, 49, 1), (10, 50, 2), (10, 40, 5), (10, 55, 0)):
        buf = torch.rand(400, generator=gen(1)).to(DEV)
        before = buf.clone()
        with pytest.raises(RuntimeError, match="overlap"):
            G.accumulate_weights(buf[50:50 + P], buf.as_strided((P,), (stride,), start), 0.5)
        assert torch.equal(buf, before)


def test_rows_moved_are_counted_before_the_first_launch():
    """The 33rd tensor goes into a second launch; that it is too large is said before the first one writes."""
    from gsr_train import compact as T
    dst = torch.full((32, 4), 9.0, device=DEV)
    small = [(dst.data_ptr(), dst[k].data_ptr(), 0, 0, 1) for k in range(32)]  # a word of padding each
    large = (1 << 52, 1 << 55, 768 * 8, 5, 0)  # 2 or more blocks a row, of 2^31 - 1 rows
    table = (T._Rows * 33)(*small, large)
    with pytest.raises(RuntimeError, match="too many rows in one call"):
        T._call(dst.device, T._lib.gsr_take_rows, 2 ** 31 - 1, 64, 33, table)
    assert (dst == 9).all()


# ---- values that the tests of the operators left out ----------------------------------------------
@pytest.mark.parametrize("n,pieces", [(5_000_011, 2), (60_000_003, 15)])
@pytest.mark.parametrize("kind", ["equal", "few", "heavy"])
def test_keep_heaviest_of_tiles_of_several_pieces(n, pieces, kind):
    """A block takes two pieces of a tile, and as many as 16-bit counts allow: 15 of 4096 rows, all of them equal."""
    import gsr_train as G
    assert min(15, max(1, (n // 4096 + 1023) // 1024)) == pieces
    g = torch.Generator(device=DEV).manual_seed(n)
    w = torch.rand(n, device=DEV, generator=g)
    if kind == "equal":
        w.fill_(0.5)
    elif kind == "few":
        w = (w * 3).floor()
    else:
        w = torch.exp(w * 40 - 20)
    for budget, recent in ((n * 2 // 3, 0), (n // 5, 12_345), (n - 1, 0)):
        old = n - recent
        order = torch.sort(w[:old], descending=True, stable=True)[1][:budget - recent]
        keep = torch.zeros(n, dtype=torch.bool, device=DEV)
        keep[order] = True
        keep[old:] = True
        want = torch.nonzero(keep).flatten().int()
        assert torch.equal(G.keep_heaviest(w, budget, recent=recent), want), budget


@pytest.mark.parametrize("degree", [0, 3])
def test_gradient_on_both_sides_of_zero(degree):
    """The constants next to -1 / (2 C_0), at the camera, where the direction and all other terms are 0: p >= 0 takes
    part.  (p = 0 itself is out of reach here: C_0 times a float is never -1/2.)"""
    import gsr_train as G
    C0 = 0.28209479177387814
    dc = torch.tensor(-0.5 / C0, dtype=torch.float64).float()
    f = torch.zeros(3, 16, 3)
    f[0, 0], f[1, 0], f[2, 0] = dc, torch.nextafter(dc, torch.tensor(-9.0)), torch.nextafter(dc, torch.tensor(9.0))
    p = 0.5 + C0 * f[:, 0].double()
    assert (p.abs() < 2.0 ** -22).all() and (p > 0).any() and (p < 0).any()
    fg = f.to(DEV).requires_grad_()
    c = G.sh_colors_quantized(torch.zeros(3, 3, device=DEV), fg, torch.zeros(3, device=DEV), degree)
    (gf,) = torch.autograd.grad(c, fg, torch.ones(3, 3, device=DEV))
    assert torch.equal(gf[:, 0].cpu() != 0, p >= 0) and (gf[:, 1:] == 0).all()


def test_degrees_of_other_integer_types_take_the_compiled_route(monkeypatch):
    """numpy integers, as a loaded scene may hold them: no slower call, and capture with gradients works."""
    import numpy as np
    import gsr_train as G
    from gsr_train import compact as T
    xyz, f, cam, up = (t.to(DEV) for t in scene(30, 9, 1, 4))
    rest = G.mx4_quantize(f.flatten(1)[:, 3:])
    want, shown = G.sh_colors_quantized(xyz, f, cam, 2), G.sh_colors(xyz, f[:, 0], rest, cam, 2)
    monkeypatch.setattr(T, "_sh_check", None)  # what the ctypes route begins with
    for degree in (np.int64(2), np.int32(2), np.uint8(2)):
        assert torch.equal(G.sh_colors_quantized(xyz, f, cam, degree), want)
        assert torch.equal(G.sh_colors(xyz, f[:, 0], rest, cam, degree), shown)
    x = xyz.clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (g,) = torch.autograd.grad(G.sh_colors_quantized(x, f, cam, np.int64(2)), x, up)
    graph.replay()
    torch.cuda.synchronize()
    (h,) = torch.autograd.grad(G.sh_colors_quantized(x, f, cam, 2), x, up)
    assert torch.equal(g, h)
