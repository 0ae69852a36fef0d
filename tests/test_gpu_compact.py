"""Compact-scene operators on the MI355X against oracle/compact_oracle.py.

Tolerances.  Codes, scales, decoded values, ids and moved rows are exact.  Colours: with u =
2^-24 (half a step of fp32 at 1), a direction's components are off by at most 6 u (the difference
1, the norm 4, the product 1), a basis value by 6 u times its slope (at most 4.9: 2.6 along the
sphere, 2.3 from the radius) plus 8 u of its own evaluation, together 37 u; 16 products added one
after the other round by 16 u of their sum.  So a channel before the clamp is off by at most
53 u < 2^-18 times (1/2 + sum |coefficient|).  Gradients of the features: 37 u of a view's |g|
plus the sum over at most 16 views: 2^-18 sum |g|.  Gradients of the positions: the basis
gradient (length at most 3.5, slope at most 15) is off by 6 * 15 + 8 * 3.5 u, the weights
(3 products) and their sum over 16 by 19 * 3.5 u, the projection and 1 / |u| by 6 * 3.5 u:
about 205 u < 2^-16 times sum_v 1 / |u_v| sum |coefficient| |g|."""
import math

import numpy as np
import pytest
import torch

from oracle import compact_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- 4-bit rows ----------------------------------------------------------------------------
def check_rows(x_gpu, what=""):
    import gsr_train as G
    q = G.mx4_quantize(x_gpu)
    codes, scales = O.mx4_quantize(x_gpu.cpu().numpy())
    assert np.array_equal(q.scales.cpu().numpy(), scales), what
    # a block with a NaN or an infinity has no codes of its own
    want = O.mx4_dequantize(codes, scales, x_gpu.shape[1])
    got = q.dequantize().cpu().numpy()
    assert got.shape == want.shape and np.array_equal(got, want, equal_nan=True), what
    assert np.array_equal(q.codes.cpu().numpy(), codes), what
    return q


@pytest.mark.parametrize("R,K", [(1, 1), (1, 45), (7, 9), (64, 24), (500, 45), (3, 32), (5, 33), (2, 64), (129, 8),
                                 (17, 31), (4, 100), (33, 3), (257, 7), (65, 63), (3, 1000)])
def test_mx4_rows(R, K):
    g = gen(R * 1000 + K)
    x = torch.randn(R, K, generator=g) * torch.exp(torch.randn(R, 1, generator=g) * 3)
    x[:: 5] = 0.0
    check_rows(x.to(DEV), f"{R}x{K}")


@pytest.mark.parametrize("R,K", [(1, 4), (2, 5), (3, 35), (1000, 9), (700, 45), (3, 1024), (7, 1025), (5, 1029), (11, 5000),
                                 (300, 34), (2049, 6), (91, 31), (40, 63)])
def test_mx4_rows_of_any_width_with_holes(R, K):
    """Rows and blocks that end inside a lane's four values; NaN and infinities here and there: only their own blocks
    read back as NaN."""
    g = gen(R * 7919 + K)
    x = torch.randn(R, K, generator=g) * torch.exp(torch.randn(R, 1, generator=g) * 3)
    hole = torch.rand(R, K, generator=g)
    x[hole < 0.01] = math.nan
    x[hole > 0.995] = -math.inf
    check_rows(x.to(DEV), f"{R}x{K}")


def test_mx4_empty():
    import gsr_train as G
    for R, K in ((0, 45), (5, 0), (0, 0)):
        q = G.mx4_quantize(torch.zeros(R, K, device=DEV))
        assert q.rows == R and q.width == K and q.dequantize().shape == (R, K)


def test_mx4_ties_scales_and_special_values():
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9999995])
    steps = torch.cat([ties, torch.nextafter(ties, torch.tensor(0.0)), torch.nextafter(ties, torch.tensor(9.0)), -ties])
    rows = []
    for e in (-149, -140, -128, -127, -126, -125, -124, -60, -1, 0, 1, 60, 120, 125):
        r = torch.ldexp(steps.double(), torch.tensor(e)).float()
        rows.append(r[torch.isfinite(r)][:38])
        rows[-1] = torch.cat([rows[-1], torch.zeros(45 - len(rows[-1]))])
    x = torch.stack(rows)
    x[:, 44] = -0.0
    check_rows(x.to(DEV))
    for bad in (float("nan"), float("inf"), -float("inf")):
        y = x.clone()
        y[3, 5] = bad     # first block of a row
        y[4, 40] = bad    # the short last one
        y[5, :32] = bad
        q = check_rows(y.to(DEV), str(bad))
        assert q.scales.cpu()[3].tolist()[0] == 255 and q.scales.cpu()[4].tolist()[1] == 255
    check_rows(torch.full((3, 45), 3.4028234e38, device=DEV))


def test_mx4_rows_apart_and_unaligned():
    x = torch.randn(300, 16, 3, generator=gen(1)).to(DEV)
    a = check_rows(x.flatten(1)[:, 3:])                     # the rest of a feature tensor: rows 48 apart
    import gsr_train as G
    b = G.mx4_quantize(x[:, 1:].flatten(1).contiguous())
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    check_rows(torch.randn(1001, generator=gen(2)).to(DEV)[1:].view(100, 10))  # starts 4 bytes off
    check_rows(torch.randn(45, 20, generator=gen(3)).to(DEV).T)               # columns: copied
    check_rows(torch.randn(1, 45, generator=gen(4)).to(DEV).expand(5, 45))    # rows that overlap: copied
    check_rows(torch.randn(40, 90, generator=gen(5)).to(DEV)[::2, ::2])


def test_mx4_rows_behind_the_last_stay():
    from gsr_train import compact as T
    x = torch.randn(10, 45, generator=gen(6)).to(DEV)
    codes = torch.full((11, 24), 0xAB, dtype=torch.uint8, device=DEV)
    scales = torch.full((11, 2), 0xCD, dtype=torch.uint8, device=DEV)
    T._call(x.device, T._lib.gsr_mx4_quantize, 10, 45, x.data_ptr(), 45, codes.data_ptr(), scales.data_ptr())
    assert (codes[10] == 0xAB).all() and (scales[10] == 0xCD).all() and not (codes[9] == 0xAB).all()
    out = torch.full((11, 45), 7.0, device=DEV)
    T._call(x.device, T._lib.gsr_mx4_dequantize, 10, 45, codes.data_ptr(), scales.data_ptr(), out.data_ptr())
    assert (out[10] == 7).all()


# ---- colours ---------------------------------------------------------------------------------
def scene(P, M, V, seed, spread=1.5):
    g = gen(seed)
    xyz = (torch.rand(P, 3, generator=g) * 2 - 1) * spread
    f = torch.randn(P, M, 3, generator=g) * 0.3
    f[:, 0] = (torch.rand(P, 3, generator=g) - 0.6) / 0.28209479177387814
    cam = torch.randn(V, 3, generator=g) * 3
    up = torch.randn(V, P, 3, generator=g)
    return xyz, f, cam, up


def decoded(f):
    P, M, _ = f.shape
    rest = f[:, 1:].reshape(P, -1).numpy()
    rest = O.mx4_dequantize(*O.mx4_quantize(rest), rest.shape[1]) if M > 1 else rest
    return torch.cat([f[:, :1], torch.from_numpy(np.ascontiguousarray(rest)).view(P, M - 1, 3)], 1)


def reference(xyz, f, cam, up, degree):
    """(colours, before the clamp, dxyz, dfeatures) in 64 bits, f decoded."""
    x, q = xyz.double().requires_grad_(), f.double().requires_grad_()
    p = O.sh_preclamp(x, q, cam, degree)
    dx, df = torch.autograd.grad(p, (x, q), up.double() * (p.detach() >= 0), materialize_grads=True)
    p = p.detach()
    return p.clamp(min=0), p, dx, df


def bounds(xyz, f, cam, up, degree):
    n = (degree + 1) ** 2
    size = 0.5 + f[:, :n].double().abs().sum(1)
    far = 1 / (xyz.double()[None] - cam.double()[:, None]).norm(dim=2)
    pull = (f[:, 1:n].double().abs().sum(1)[None] * up.double().abs()).sum(2)
    return (2.0 ** -18 * size[None], 2.0 ** -18 * up.double().abs().sum(0)[:, None],
            2.0 ** -16 * (far * pull).sum(0)[:, None] + 1e-30)


@pytest.mark.parametrize("P", [1, 2, 63, 64, 65, 255, 256, 257, 1003])
@pytest.mark.parametrize("M,degree,V", [(1, 0, 1), (4, 0, 2), (4, 1, 1), (9, 1, 3), (9, 2, 1), (16, 3, 1), (16, 3, 5),
                                        (16, 2, 16), (16, 0, 1), (12, 2, 2), (5, 1, 1)])
def test_colors_and_gradients(P, M, degree, V):
    import gsr_train as G
    xyz, f, cam, up = scene(P, M, V, P * 100 + M + degree)
    q = decoded(f)
    want, _, dx, df = reference(xyz, q, cam, up, degree)
    tc, tf, tx = bounds(xyz, q, cam, up, degree)
    x, fg = xyz.to(DEV).requires_grad_(), f.to(DEV).requires_grad_()
    c = G.sh_colors_quantized(x, fg, cam.to(DEV), degree)
    assert c.shape == (V, P, 3) and (c >= 0).all()
    assert ((c.detach().cpu().double() - want).abs() <= tc).all()
    gx, gf = torch.autograd.grad(c, (x, fg), up.to(DEV))
    assert ((gf.cpu().double() - df).abs() <= tf).all()
    assert ((gx.cpu().double() - dx).abs() <= tx).all()
    assert (gf[:, (degree + 1) ** 2:] == 0).all()
    # the same from codes made beforehand: the same bits, and gradients of positions and constants
    rest = G.mx4_quantize(f.to(DEV).flatten(1)[:, 3:])
    dc = f[:, :1].to(DEV).contiguous().requires_grad_()
    c2 = G.sh_colors(x, dc, rest, cam.to(DEV), degree)
    assert torch.equal(c2, c)
    hx, hd = torch.autograd.grad(c2, (x, dc), up.to(DEV))
    assert torch.equal(hx, gx) and torch.equal(hd, gf[:, :1])
    # a constant that is a view of the features, and one camera without the views axis
    c3 = G.sh_colors(x, fg.detach()[:, 0], rest, cam[0].to(DEV), degree)
    assert c3.shape == (P, 3) and torch.equal(c3, c[0])
    (only_x,) = torch.autograd.grad(c3, x, up[0].to(DEV))
    assert only_x.shape == (P, 3)
    (only_f,) = torch.autograd.grad(G.sh_colors_quantized(x.detach(), fg, cam.to(DEV), degree), fg, up.to(DEV))
    assert torch.equal(only_f, gf)


def test_gradient_against_differences():
    """Directional differences of the 64-bit colours (away from the clamp) against the kernel's
    gradients: central differences with h = 1e-4 are off by h^2 / 6 times a third derivative
    (at most 200 times the scale of the bounds)."""
    import gsr_train as G
    P, V, degree = 50, 2, 3
    xyz, f, cam, up = scene(P, 16, V, 77)
    q = decoded(f)
    _, p, _, _ = reference(xyz, q, cam, up, degree)
    up = torch.where(p.abs() < 0.02, torch.zeros_like(p), up.double()).float()
    x, fg = xyz.to(DEV).requires_grad_(), f.to(DEV).requires_grad_()
    gx, gf = torch.autograd.grad(G.sh_colors_quantized(x, fg, cam.to(DEV), degree), (x, fg), up.to(DEV))
    _, tf, tx = bounds(xyz, q, cam, up, degree)
    h = 1e-4

    def value(dx, dq):
        c = O.sh_preclamp(xyz.double() + dx, q.double() + dq, cam, degree).clamp(min=0)
        return (c * up.double()).sum((0, 2))

    for axis in range(3):
        e = torch.zeros(3, dtype=torch.float64)
        e[axis] = h
        d = (value(e, 0) - value(-e, 0)) / (2 * h)
        assert ((gx.cpu().double()[:, axis] - d).abs() <= (tx * (1 + 200 * h * h / 6 * 2.0 ** 16))[:, 0]).all()
    for k, ch in ((0, 0), (1, 2), (7, 1), (15, 0)):
        e = torch.zeros(16, 3, dtype=torch.float64)
        e[k, ch] = h
        d = (value(0, e) - value(0, -e)) / (2 * h)  # linear: the difference itself is exact to 1e-11
        assert ((gf.cpu().double()[:, k, ch] - d).abs() <= tf[:, 0, ch] + 1e-10).all()


def test_gradient_next_to_the_clamp():
    """Values before the clamp within a few units of fp32 around zero: which channels get a
    gradient is decided as in 64 bits."""
    import gsr_train as G
    P = 4096
    xyz, f, cam, up = scene(P, 16, 1, 5)
    f[:, 1:] *= 0.2
    for _ in range(2):  # move the constant to where the value is zero, then a few units off
        q = decoded(f)
        p = O.sh_preclamp(xyz, q, cam, 3)[0]
        f[:, 0] = (f[:, 0].double() - p / 0.28209479177387814).float()
    off = torch.randint(-3, 4, (P, 3), generator=gen(6))
    bits = f[:, 0].contiguous().view(torch.int32) + off.int()
    f[:, 0] = bits.view(torch.float32)
    p = O.sh_preclamp(xyz, decoded(f), cam, 3)[0]
    assert (p.abs() < 3e-6).all() and (p > 0).sum() > 1000 and (p < 0).sum() > 1000
    fg = f.to(DEV).requires_grad_()
    (gf,) = torch.autograd.grad(G.sh_colors_quantized(xyz.to(DEV), fg, cam[0].to(DEV), 3), fg,
                                torch.ones(P, 3, device=DEV))
    assert torch.equal(gf[:, 0].cpu() != 0, p >= 0)
    # exactly at zero (degree 0 has no rounding that matters: a constant of 0 and -0.5 / Y_0 below it)
    z = torch.zeros(2, 1, 3)
    z[1] = -4.0
    zg = z.to(DEV).requires_grad_()
    c = G.sh_colors_quantized(torch.zeros(2, 3, device=DEV), zg, torch.ones(3, device=DEV), 0)
    assert c.tolist() == [[0.5] * 3, [0.0] * 3]


def test_colors_at_the_camera_far_away_and_not_finite():
    import gsr_train as G
    M = 16
    xyz = torch.tensor([[1.0, 2, 3], [1, 2, 3 + 1e-6], [3e5, -2e6, 1e6], [1e20, -2e20, 3e20], [1e-30, 2e-30, -1e-30],
                        [1, 2, 3]])
    f = torch.randn(6, M, 3, generator=gen(8)) * 0.1
    f[5, 3, 1] = float("nan")
    cam = torch.tensor([[1.0, 2, 3], [0, 0, 0]])
    q = decoded(f)
    up = torch.randn(2, 6, 3, generator=gen(9))
    x, fg = xyz.to(DEV).requires_grad_(), f.to(DEV).requires_grad_()
    c = G.sh_colors_quantized(x, fg, cam.to(DEV), 3)
    gx, gf = torch.autograd.grad(c, (x, fg), up.to(DEV))
    want = O.sh_preclamp(xyz, q, cam, 3).clamp(min=0)
    ok = slice(0, 5)
    tc = 2.0 ** -18 * (0.5 + q.double().abs().sum(1))[None]
    assert ((c.detach().cpu().double() - want).abs() <= tc)[:, ok].all()
    assert torch.isnan(c[:, 5]).all() and torch.isnan(want[:, 5]).all()  # the NaN took the first block: all channels
    assert torch.isfinite(gx[ok]).all() and torch.isfinite(gf[:5]).all()
    # at the camera: only the other view gives the position a gradient
    (g1,) = torch.autograd.grad(G.sh_colors_quantized(x, fg.detach(), cam[1:].to(DEV), 3), x, up[1:].to(DEV))
    (g0,) = torch.autograd.grad(G.sh_colors_quantized(x, fg.detach(), cam[:1].to(DEV), 3), x, up[:1].to(DEV))
    assert (g0[0] == 0).all() and torch.equal(gx[0], g1[0])


def test_colors_empty_and_not_contiguous():
    import gsr_train as G
    c = G.sh_colors_quantized(torch.zeros(0, 3, device=DEV), torch.zeros(0, 16, 3, device=DEV),
                              torch.zeros(2, 3, device=DEV), 3)
    assert c.shape == (2, 0, 3)
    xyz, f, cam, up = scene(100, 16, 2, 3)
    a = G.sh_colors_quantized(xyz.to(DEV), f.to(DEV), cam.to(DEV), 3)
    xt = xyz.T.contiguous().to(DEV).T
    ft = f.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    x, fg = xt.requires_grad_(), ft.requires_grad_()
    b = G.sh_colors_quantized(x, fg, cam.to(DEV), 3)
    assert torch.equal(a, b)
    upt = up.permute(0, 2, 1).contiguous().permute(0, 2, 1).to(DEV)
    gx, gf = torch.autograd.grad(b, (x, fg), upt)
    x2, f2 = xyz.to(DEV).requires_grad_(), f.to(DEV).requires_grad_()
    hx, hf = torch.autograd.grad(G.sh_colors_quantized(x2, f2, cam.to(DEV), 3), (x2, f2), up.to(DEV))
    assert torch.equal(gx, hx) and torch.equal(gf, hf)
    # a gradient that is one number broadcast
    (gs,) = torch.autograd.grad(G.sh_colors_quantized(x2, f2, cam.to(DEV), 3).sum(), f2)
    (ho,) = torch.autograd.grad(G.sh_colors_quantized(x2, f2, cam.to(DEV), 3), f2, torch.ones(2, 100, 3, device=DEV))
    assert torch.equal(gs, ho)


def both_routes(monkeypatch):
    """The C++ host binding and ctypes in turn."""
    from gsr_train import compact as T
    assert T._HOST is not None, "gsr_host not built (__graft_entry__.build())"
    yield "host"
    monkeypatch.setattr(T, "_HOST", None)
    yield "ctypes"


def test_both_host_routes_give_the_same(monkeypatch):
    import gsr_train as G
    xyz, f, cam, up = scene(3000, 16, 3, 12)
    w = torch.exp(torch.randn(50_000, generator=gen(1))).to(DEV)
    rows = [torch.randn(50_000, k, generator=gen(k)).to(DEV) for k in (1, 3, 48)]
    got = {}
    for route in both_routes(monkeypatch):
        x, fg = xyz.to(DEV).requires_grad_(), f.to(DEV).requires_grad_()
        q = G.mx4_quantize(fg.detach().flatten(1)[:, 3:])
        dc = f[:, 0].to(DEV).requires_grad_()
        a = G.sh_colors_quantized(x, fg, cam.to(DEV), 3)
        b = G.sh_colors(x, dc, q, cam.to(DEV), 3)
        assert a.requires_grad and b.requires_grad
        with torch.no_grad():
            c = G.sh_colors_quantized(x, fg, cam.to(DEV), 3)
        assert not c.requires_grad and not G.sh_colors(x.detach(), dc.detach(), q, cam.to(DEV), 3).requires_grad
        ids = G.keep_heaviest(w, [100, 20_000], [(0, 5000), (5000, 50_000)], 7)
        got[route] = [q.codes, q.scales, q.dequantize(), a, b, c, ids, *G.take_rows(ids, rows),
                      *torch.autograd.grad(a, (x, fg), up.to(DEV)), *torch.autograd.grad(b, (x, dc), up.to(DEV))]
        with pytest.raises(RuntimeError, match="tensors.1. must be"):
            G.take_rows(ids, [rows[0], rows[1].double()])
        with pytest.raises(RuntimeError, match="out.0. must be"):
            G.take_rows(ids, [rows[0]], out=[rows[1]])
        with pytest.raises(RuntimeError, match="contiguous"):
            G.take_rows(ids, [rows[2][:, ::2]])
    for a, b in zip(got["host"], got["ctypes"]):
        assert a.shape == b.shape and torch.equal(a, b)


def test_colors_double_backward_is_refused(monkeypatch):
    for _ in both_routes(monkeypatch):
        check_double_backward()


def check_double_backward():
    import gsr_train as G
    xyz, f, cam, up = scene(10, 4, 1, 3)
    x = xyz.to(DEV).requires_grad_()
    c = G.sh_colors_quantized(x, f.to(DEV), cam.to(DEV), 1)
    (gx,) = torch.autograd.grad(c.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gx.sum().backward()


# ---- eviction ----------------------------------------------------------------------------------
def check_keep(w, budgets, groups=None, recent=0):
    import gsr_train as G
    from gsr_train.compact import _keep_groups
    ids = G.keep_heaviest(w.to(DEV), budgets, groups, recent)
    want = O.keep_heaviest(w.numpy().reshape(-1), _keep_groups("t", w.numel(), budgets, groups, recent))
    assert ids.dtype == torch.int32 and np.array_equal(ids.cpu().numpy(), want)
    return ids


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 1000, 4095, 4096, 4097, 16384, 16385, 40001])
@pytest.mark.parametrize("kind", ["heavy", "equal", "two", "special", "signed"])
def test_keep_heaviest(n, kind):
    g = gen(n)
    w = torch.exp(torch.randn(n, generator=g) * 3)
    if kind == "equal":
        w[:] = 0.25
    elif kind == "two":
        w = torch.where(torch.rand(n, generator=g) < 0.4, torch.tensor(0.0), torch.tensor(-0.0)) + \
            (torch.rand(n, generator=g) < 0.3).float()
    elif kind == "special":
        pick = torch.randint(0, 8, (n,), generator=g)
        for k, v in enumerate((float("nan"), float("inf"), -float("inf"), 1e-45, -0.0)):
            w[pick == k] = v
        w[pick == 7] = -float("nan")
    elif kind == "signed":
        w = torch.randn(n, generator=g)
    for budget in sorted({0, 1, n // 3, n // 2, n - 1, n, n + 5}):
        check_keep(w, budget)
        check_keep(w, budget, recent=n // 10)
    check_keep(w, n // 2, recent=n)


def test_keep_heaviest_groups():
    g = gen(3)
    w = torch.exp(torch.randn(100_000, generator=g))
    w[torch.rand(100_000, generator=g) < 0.3] = 0.0
    groups = [(0, 7), (7, 7), (10, 20_000), (20_000, 20_001), (20_001, 60_000), (70_000, 99_999)]
    check_keep(w, 5000, groups)
    check_keep(w, [0, 3, 1, 0, 39_999, 12_345], groups, recent=[0, 1, 1, 1, 500, 12_345])
    check_keep(w, [7, 3, 30_000, 1, 0, 29_999], groups, 4)
    check_keep(w, 100, [(k * 1500, k * 1500 + 1500 - k) for k in range(64)], 3)  # as many as a call takes
    check_keep(w, 10, [])
    check_keep(torch.zeros(0), 10)
    check_keep(w[:5000].view(5000, 1), 77)  # [P, 1], as the model holds them


@pytest.mark.parametrize("n", [4100, 8191, 8192, 8193, 12_287, 12_288, 12_289])
def test_keep_heaviest_runs_of_equal_weights(n):
    """Runs that fill a thread's keys or end inside them, at the sizes where a thread takes more."""
    g = gen(n)
    for run in (4, 7, 16, 1000):
        w = torch.exp(torch.randn(n // run + 1, generator=g)).repeat_interleave(run)[:n].contiguous()
        for budget in (run, n // 2, n // 2 + 1, n - 1):
            check_keep(w, budget)
            check_keep(w, budget, recent=run // 2)
    check_keep(torch.full((n,), float("nan")), n // 3)


@pytest.mark.parametrize("kind", ["heavy", "equal", "whole"])
def test_keep_heaviest_of_many_rows(kind):
    """9M rows (a block takes two pieces of a tile) and 17M (three): in one group, and in groups of unequal size whose
    ends lie inside a piece."""
    g = gen(9)
    n = 9_000_001 if kind != "whole" else 17_000_003
    w = torch.exp(torch.randn(n, generator=g) * 2)
    if kind == "equal":
        w[:] = 0.5
    elif kind == "whole":  # few values, most of them often
        w = (w * 4).floor()
    import gsr_train as G
    w = w.to(DEV)

    def want(groups, budget, recent):
        keep = torch.zeros(n, dtype=torch.bool, device=DEV)
        for (a, b), r in zip(groups, recent):
            k = min(budget, b - a)
            r = min(r, k)
            keep[a + torch.sort(w[a:b - r], descending=True, stable=True)[1][:k - r]] = True
            keep[b - r:b] = True
        return torch.nonzero(keep).flatten().int()

    assert torch.equal(G.keep_heaviest(w, n * 3 // 5), want([(0, n)], n * 3 // 5, [0]))
    groups, recent = [(0, 5000), (5000, 4_105_001), (4_200_000, 4_208_193), (4_208_193, n)], [0, 100_000, 5, 9]
    assert torch.equal(G.keep_heaviest(w, n // 3, groups, recent), want(groups, n // 3, recent))


def test_keep_heaviest_twice_at_once_and_on_other_streams():
    import gsr_train as G
    w = [torch.exp(torch.randn(200_000, generator=gen(k))).to(DEV) for k in range(4)]
    want = [G.keep_heaviest(x, 50_000) for x in w]
    streams = [torch.cuda.Stream() for _ in w]
    got = []
    for s, x in zip(streams, w):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(G.keep_heaviest(x * 1.0, 50_000))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("K", [0, 1, 63, 64, 65, 1000, 5000])
def test_take_rows(K):
    import gsr_train as G
    g = gen(K)
    P = 3001
    ids = torch.randint(0, P, (K,), generator=g, dtype=torch.int32)  # any order, the same row twice
    t = [torch.randn(P, k, generator=g) for k in (1, 2, 3, 4, 5, 7, 8, 12, 45, 48)]
    t += [torch.randn(P, 16, 3, generator=g), torch.randn(P, generator=g),
          torch.randint(-9, 9, (P, 2), generator=g, dtype=torch.int32), torch.zeros(P, 0)]
    t += [torch.randn(P, 3, generator=g) for _ in range(30)]  # more than one launch takes
    t.append(torch.randn(P * 3 + 1, generator=g)[1:].view(P, 3))
    dev = [x.to(DEV) for x in t[:-1]] + [t[-1].new_empty(P * 3 + 1).to(DEV)[1:].view(P, 3).copy_(t[-1])]
    got = G.take_rows(ids.to(DEV), dev)
    for x, y in zip(t, got):
        assert y.dtype == x.dtype and torch.equal(y.cpu(), x[ids.long()])
    out = [torch.full_like(y, 5) for y in got]
    assert all(a is b for a, b in zip(G.take_rows(ids.to(DEV), dev, out=out), out))
    assert all(torch.equal(a, b) for a, b in zip(out, got))


def test_take_rows_refuses_an_output_that_overlaps(monkeypatch):
    import gsr_train as G
    x = torch.randn(10, 3, device=DEV)
    ids = torch.arange(10, dtype=torch.int32, device=DEV)
    for _ in both_routes(monkeypatch):
        with pytest.raises(RuntimeError, match="overlaps"):
            G.take_rows(ids, [x], out=[x])
        with pytest.raises(RuntimeError, match="overlaps"):
            G.take_rows(ids, [x, x.clone()], out=[torch.empty_like(x), x])


def test_take_rows_refuses_more_ids_than_an_int_counts():
    import gsr_train as G
    with pytest.raises(RuntimeError, match="2\\^31"):
        G.take_rows(torch.empty(2 ** 31, dtype=torch.int32, device=DEV), [torch.zeros(3, 0, device=DEV)])


def test_take_rows_of_ids_outside():
    import gsr_train as G
    x = torch.randn(10, 3, device=DEV)
    ids = torch.tensor([3, -1, 10, 2 ** 31 - 1, 0], dtype=torch.int32, device=DEV)
    y, z = G.take_rows(ids, [x, torch.zeros(0, 3, device=DEV)])
    assert torch.equal(y[0], x[3]) and torch.equal(y[4], x[0]) and (y[1:4] == 0).all() and (z == 0).all()


@pytest.mark.parametrize("width", [6, 9, 10, 14, 15, 16, 27, 30, 768, 770, 2304, 2306, 2307, 2308])
def test_take_rows_of_every_unit(width):
    """Rows of 16-, 12-, 8- and 4-byte units, from memory that starts at any word and to memory that does."""
    import gsr_train as G
    K, P = 1000, 700
    ids = torch.randint(-2, P + 2, (K,), generator=gen(width), dtype=torch.int32).to(DEV)
    inside = ((ids >= 0) & (ids < P)).view(K, 1)
    for lead in range(4):
        x = torch.randn(P * width + lead, generator=gen(3)).to(DEV)[lead:].view(P, width)
        want = torch.where(inside, x[ids.clamp(0, P - 1).long()], torch.zeros((), device=DEV))
        assert torch.equal(G.take_rows(ids, [x])[0], want)
        buf = torch.full((K * width + lead + 1,), 9.0, device=DEV)
        out = buf[lead:-1].view(K, width)
        G.take_rows(ids, [x], out=[out])
        assert torch.equal(out, want) and (buf[:lead] == 9).all() and buf[-1] == 9


def test_take_rows_wide_and_padded():
    """Rows wider than a block's span, and the words behind a destination's last row."""
    from gsr_train import compact as T
    ids = torch.randint(0, 50, (40,), generator=gen(1), dtype=torch.int32).to(DEV)
    for width in (1023, 1024, 1025, 1500, 4096, 4100, 9001):
        x = torch.randn(50, width, generator=gen(width)).to(DEV)
        assert torch.equal(T.take_rows(ids, [x])[0], x[ids.long()]), width
    for K, width, pad in ((40, 3, 7), (0, 3, 70), (40, 0, 300), (21, 48, 0), (1, 12, 2000)):
        x = torch.randn(50, width, generator=gen(2)).to(DEV)
        buf = torch.full((K * width + pad + 5,), 9.0, device=DEV)
        table = (T._Rows * 1)((x.data_ptr(), buf.data_ptr(), width, 50, pad))
        T._call(x.device, T._lib.gsr_take_rows, K, ids.data_ptr(), 1, table)
        assert torch.equal(buf[:K * width].view(K, width), x[ids[:K].long()])
        assert (buf[K * width:K * width + pad] == 0).all() and (buf[K * width + pad:] == 9).all()


def test_accumulate_weights():
    import gsr_train as G
    w = torch.randn(1001, 3, generator=gen(1)).to(DEV)
    acc = torch.randn(1001, 1, generator=gen(2)).to(DEV)
    want = (acc[:, 0].double() * 0.9 + w[:, 1].double())
    G.accumulate_weights(acc, w[:, 1], 0.9)
    # one product (or none, fused) and one sum; 0.9 itself is rounded to fp32 once
    assert ((acc[:, 0].double() - want).abs() <= 2.0 ** -22 * (want.abs() + w[:, 1].double().abs() + 1)).all()


# ---- the model -----------------------------------------------------------------------------------
class Args:
    position_lr_init, position_lr_final, position_lr_delay_mult, position_lr_max_steps = 1.6e-4, 1.6e-6, 0.01, 30000
    feature_lr, opacity_lr, segment_lr, scaling_lr, rotation_lr, percent_dense = 0.0025, 0.05, 0.05, 0.005, 0.001, 0.01


def model(P=3000, degree=3, seed=0):
    from gsr_tools.scene import synthetic_scene
    from gsr_train import GaussianModel
    s = synthetic_scene(P, sh_degree=degree, seed=seed, log_scale=-3.0)
    m = GaussianModel(degree, device=DEV)
    m.create_from_tensors(s.means3D, s.shs[:, :1], s.shs[:, 1:], torch.logit(s.opacities), torch.logit(s.segments),
                          torch.log(s.scales), s.rotations)
    m.spatial_lr_scale = 1.0
    m.training_setup(Args)
    m.active_sh_degree = degree
    g = torch.Generator(device=DEV).manual_seed(seed)
    m.optimizer.exp_avg.normal_(generator=g)
    m.optimizer.exp_avg_sq.uniform_(generator=g)
    m.xyz_gradient_accum.uniform_(generator=g)
    m.denom.uniform_(generator=g)
    m.max_radii2D.uniform_(generator=g)
    m.contribution.uniform_(generator=g)
    return m


def camera(k=0, W=160, H=120):
    from gsr_tools.scene import orbit_camera
    return orbit_camera(k, W, H, 150.0)


@pytest.mark.parametrize("budget,recent,groups", [(1000, 0, None), (2500, 700, None), ([500, 900], [100, 0], [(0, 1000), (1000, 3000)]),
                                                  (5000, 0, None), (0, 0, None)])
def test_model_evict_equals_prune_points(budget, recent, groups):
    """The rows that stay, their moments and statistics are those of prune_points with the
    complement's mask."""
    from gsr_train.compact import _keep_groups
    a, b = model(), model()
    ids = O.keep_heaviest(a.contribution.cpu().numpy().reshape(-1), _keep_groups("t", 3000, budget, groups, recent))
    got, ranges = a.evict(budget, recent=recent, groups=groups)
    assert np.array_equal(got.cpu().numpy(), ids)
    assert ranges[-1][1] == a.num_points == len(ids) and ranges[0][0] == 0
    mask = torch.ones(3000, dtype=torch.bool)
    mask[torch.from_numpy(ids).long()] = False
    b.prune_points(mask.to(DEV))
    for x, y in ((a._arena.data, b._arena.data), (a.optimizer.exp_avg, b.optimizer.exp_avg),
                 (a.optimizer.exp_avg_sq, b.optimizer.exp_avg_sq), (a.xyz_gradient_accum, b.xyz_gradient_accum),
                 (a.denom, b.denom), (a.max_radii2D, b.max_radii2D), (a.contribution, b.contribution),
                 (a.get_opacity, b.get_opacity), (a.get_rotation, b.get_rotation)):
        assert x.shape == y.shape and torch.equal(x, y)
    assert a.optimizer.param_groups[0]["params"][0].shape == (len(ids), 3)


def test_blend_weights_sum_to_the_alpha_image():
    """Sum over the Gaussians of alpha * T = sum over the pixels of the alpha image; each side
    adds about 2e4 terms in fp32, some pairwise: 2^-24 * 2e4 of the sum at most."""
    from gsr_tools.train_demo import blend_weights, render
    m, cam = model(), camera()
    w = blend_weights(cam, m)
    with torch.no_grad():
        pkg = render(cam, m, torch.zeros(3, device=DEV))
    assert w.shape == (3000,) and (w >= 0).all() and (w[pkg["radii"] == 0] == 0).all()
    a, b = float(w.double().sum()), float(pkg["alpha"].double().sum())
    assert b > 100 and abs(a - b) <= 2.0 ** -24 * 2e4 * b
    before = m.contribution.clone()
    m.add_contribution_stats(w, decay=0.5)
    assert torch.allclose(m.contribution, before * 0.5 + w[:, None], rtol=2.0 ** -22, atol=2.0 ** -22)


def test_compact_scene_shows_what_the_model_trained():
    """Densify, evict to a budget, train with 4-bit coefficients, store: the stored scene's
    image is the model's, bit for bit, and gradients reached every block."""
    from gsr_tools.train_demo import OptArgs, blend_weights, render, train
    from gsr_train import CompactGaussians
    m = model()
    bg = torch.zeros(3, device=DEV)
    cams = [camera(k) for k in range(3)]
    with torch.no_grad():
        targets = [render(c, m, bg)["render"].clone() for c in cams]

    class Opt(OptArgs):
        densify_from_iter, densification_interval, densify_grad_threshold = 2, 4, 1e-7
        gaussian_budget = 2000

    m.feature_bits = 4
    sizes = []
    losses = train(m, cams, targets, 9, opt=Opt, log=lambda it, loss, n: sizes.append(n),
                   generator=torch.Generator(device=DEV).manual_seed(1))
    assert all(np.isfinite(losses)) and sizes[2] == 3000 and sizes[-1] == 2000 and m.num_points == 2000
    pkg = render(cams[0], m, bg)
    (pkg["render"] - targets[0]).abs().mean().backward()
    spec = m._spec
    for name in ("xyz", "features", "opacity", "scaling", "rotation"):
        assert float(spec.block(m._arena.grad, name).abs().sum()) > 0, name
    small = m.compact()
    with torch.no_grad():
        image = render(cams[1], m, bg)["render"]
        assert torch.equal(render(cams[1], small, bg)["render"], image)
        copy = CompactGaussians.from_state_dict({k: v.cpu() if isinstance(v, torch.Tensor) else v
                                                 for k, v in small.state_dict().items()}, DEV)
        assert torch.equal(render(cams[1], copy, bg)["render"], image)
        assert torch.equal(blend_weights(cams[1], small), blend_weights(cams[1], m))
        cam3 = torch.stack([c.camera_center for c in cams]).to(DEV)
        assert torch.equal(small.get_colors(cam3), m.get_colors(cam3))
    assert small.nbytes == 2000 * (12 + 12 + 24 + 2 + 4 + 12 + 16 + 8)
    want = decoded(m.get_features.detach().cpu())
    assert torch.equal(small.get_features.cpu(), want)


def test_render_in_4_bits_is_close_to_32():
    """A coefficient is off by at most a third of itself (5 rounds to 4 or 6, 8 - to 6) or a quarter step of
    its block: the colours by what that makes of the coefficients, and the image, a convex mix, by no more."""
    from gsr_tools.train_demo import render
    m, cam = model(), camera()
    bg = torch.zeros(3, device=DEV)
    f = m.get_features.detach()
    with torch.no_grad():
        a = render(cam, m, bg)["render"]
        m.feature_bits = 4
        b = render(cam, m, bg)["render"]
    err = (decoded(f.cpu()) - f.cpu()).abs().sum(1).max()  # |Y| < 1
    assert 0 < float((a - b).abs().max()) <= float(err) + 1e-4


def test_sh0_model_has_no_codes():
    from gsr_tools.train_demo import render
    m, cam = model(degree=0), camera()
    bg = torch.zeros(3, device=DEV)
    with torch.no_grad():
        a = render(cam, m, bg)["render"]
        m.feature_bits = 4
        b = render(cam, m, bg)["render"]
        c = render(cam, m.compact(), bg)["render"]
    assert torch.equal(b, c) and torch.allclose(a, b, atol=1e-5)


def test_models_without_gaussians_or_optimizer():
    from gsr_train import GaussianModel
    for degree in (0, 3):
        e = GaussianModel(degree, device=DEV)
        e.feature_bits = 4
        small = e.compact()
        cam = torch.zeros(3, device=DEV)
        assert small.num_points == 0 and small.get_features.shape == (0, (degree + 1) ** 2, 3)
        assert small.get_colors(cam).shape == (0, 3) and e.get_colors(cam).shape == (0, 3)
        ids, ranges = e.evict(5)
        assert ids.numel() == 0 and ranges == [(0, 0)] and e.num_points == 0
    m = model(degree=1)
    m.optimizer = None  # a scene that was only loaded
    want = O.keep_heaviest(m.contribution.cpu().numpy().reshape(-1), [(0, 3000, 100, 10)])
    xyz = m._xyz.clone()
    ids, _ = m.evict(100, recent=10)
    assert np.array_equal(ids.cpu().numpy(), want) and torch.equal(m._xyz, xyz[ids.long()])
    m2 = model(degree=0)
    assert m2.compact().get_features.shape == (3000, 1, 3)


def test_step_after_eviction():
    """The optimizer goes on with the moments of the Gaussians that stayed."""
    a, b = model(), model()
    ids, _ = a.evict(1200)
    g = torch.randn(a._spec.total, generator=gen(4)).to(DEV)
    full = torch.zeros(b._spec.total, device=DEV)
    for name in ("xyz", "features", "opacity", "scaling", "rotation", "segment"):
        b._spec.block(full, name)[ids.long()] = a._spec.block(g, name)
    for m, grad in ((a, g), (b, full)):
        m._arena.grad = grad
        m.optimizer.step()
    for name in ("xyz", "features", "opacity", "scaling", "rotation", "segment"):
        assert torch.equal(a._spec.block(a._arena.data, name), b._spec.block(b._arena.data, name)[ids.long()]), name


@pytest.mark.parametrize("M,degree", [(16, 3), (16, 0), (9, 2), (4, 1)])
def test_colors_of_large_calls_equal_those_of_parts(M, degree):
    """120k Gaussians, 16 views: 23 MB of colours (and 23 of gradients of the features at M = 16), whose rows and colours
    go past the caches; the parts of 7.7 MB go through them."""
    import gsr_train as G
    P, V = 120_001, 16
    xyz, f, cam, up = (t.to(DEV) for t in scene(P, M, V, 77))
    q = G.mx4_quantize(f.flatten(1)[:, 3:])
    dc = f[:, 0].contiguous()
    leaves = [t.clone().requires_grad_() for t in (xyz, f, dc)]
    shown = G.sh_colors(xyz, dc, q, cam, degree)
    held = G.sh_colors(leaves[0], leaves[2], q, cam, degree)
    trained = G.sh_colors_quantized(leaves[0], leaves[1], cam, degree)
    gd = torch.autograd.grad(held, (leaves[0], leaves[2]), up)
    gt = torch.autograd.grad(trained, leaves[:2], up)
    assert torch.equal(shown, held) and torch.equal(shown, trained)
    for a in range(0, P, 40_000):
        part = slice(a, min(P, a + 40_000))
        x, g = xyz[part].clone().requires_grad_(), f[part].clone().requires_grad_()
        rows = G.MX4Rows(q.codes[part].contiguous(), q.scales[part].contiguous(), q.width)
        d = dc[part].clone().requires_grad_()
        u = up[:, part].contiguous()
        assert torch.equal(shown[:, part], G.sh_colors(x.detach(), d.detach(), rows, cam, degree))
        c = G.sh_colors(x, d, rows, cam, degree)
        assert torch.equal(shown[:, part], c)
        for have, want in zip(gd, torch.autograd.grad(c, (x, d), u)):
            assert torch.equal(have[part], want)
        c = G.sh_colors_quantized(x, g, cam, degree)
        assert torch.equal(shown[:, part], c)
        for have, want in zip(gt, torch.autograd.grad(c, (x, g), u)):
            assert torch.equal(have[part], want)


# ---- offsets past 32 bits --------------------------------------------------------------------------
def test_offsets_past_32_bits():
    """45M Gaussians at degree 3: 2.16e9 feature values, 8.6 GB.  All zero but for the last rows and a few
    others, which have to come out as in a tensor of their own."""
    import gsr_train as G
    P, tail = 45_000_000, 300
    some = torch.cat([torch.arange(50), torch.arange(22_369_600, 22_369_700), torch.arange(P - tail, P)])
    xyz, f, cam, up = scene(len(some), 16, 1, 31)
    at = some.to(DEV)
    x = torch.zeros(P, 3, device=DEV)
    x[at] = xyz.to(DEV)
    feat = torch.zeros(P, 16, 3, device=DEV)
    feat[at] = f.to(DEV)
    q, want = G.mx4_quantize(feat.flatten(1)[:, 3:]), G.mx4_quantize(f.to(DEV).flatten(1)[:, 3:])
    assert torch.equal(q.codes[at], want.codes) and torch.equal(q.scales[at], want.scales)
    assert int(q.codes.ne(0).any(1).sum()) == int(want.codes.ne(0).any(1).sum())
    back = q.dequantize()
    assert torch.equal(back[at], want.dequantize())
    del back
    x.requires_grad_()
    feat.requires_grad_()
    sx, sf = xyz.to(DEV).requires_grad_(), f.to(DEV).requires_grad_()
    c, s = G.sh_colors_quantized(x, feat, cam[0].to(DEV), 3), G.sh_colors_quantized(sx, sf, cam[0].to(DEV), 3)
    assert torch.equal(c[at], s)
    assert torch.equal(G.sh_colors(x.detach(), feat.detach()[:, 0], q, cam[0].to(DEV), 3)[at], s)
    g = torch.zeros(P, 3, device=DEV)
    g[at] = up[0].to(DEV)
    gx, gf = torch.autograd.grad(c, (x, feat), g)
    hx, hf = torch.autograd.grad(s, (sx, sf), up[0].to(DEV))
    assert torch.equal(gx[at], hx) and torch.equal(gf[at], hf)
    assert int(gf.flatten(1).ne(0).any(1).sum()) == int(hf.flatten(1).ne(0).any(1).sum())
    del c, gx, gf, g, q
    w = torch.zeros(P, device=DEV)
    w[at] = torch.rand(len(some), generator=gen(2)).to(DEV) + 1
    ids = G.keep_heaviest(w, len(some))
    assert torch.equal(ids.cpu().long(), some)
    # many rows out: the kept ones and everything behind the first 100
    ids = torch.arange(100, P, dtype=torch.int32, device=DEV)
    (rows,) = G.take_rows(ids, [feat.detach()])
    assert torch.equal(rows[-tail:], f[-tail:].to(DEV)) and int(rows[:1000].ne(0).sum()) == 0
    assert torch.equal(rows[22_369_500:22_369_600], f[50:150].to(DEV))


# ---- graphs --------------------------------------------------------------------------------------
def test_captured_and_replayed():
    """One graph of eviction and of a forward and backward pass, replayed on new inputs with eager work
    between the replays."""
    import gsr_train as G
    xyz, f, cam, up = scene(5000, 16, 2, 21)
    x, fg = xyz.to(DEV).requires_grad_(), f.to(DEV).requires_grad_()
    cam, up = cam.to(DEV), up.to(DEV)
    w = torch.exp(torch.randn(30_000, generator=gen(2))).to(DEV)
    rows = torch.randn(30_000, 3, generator=gen(3)).to(DEV)

    def step():
        c = G.sh_colors_quantized(x, fg, cam, 3)
        gx, gf = torch.autograd.grad(c, (x, fg), up)
        ids = G.keep_heaviest(w, 12_345, recent=100)
        return c.detach(), gx, gf, ids, G.take_rows(ids, [rows])[0], G.mx4_quantize(rows).dequantize()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for k in range(4):
        with torch.no_grad():
            x.add_(0.01)
            fg.mul_(1.05)
            w.copy_(torch.exp(torch.randn(30_000, generator=gen(10 + k))))
            rows.mul_(-1.1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(static, step()):
            assert torch.equal(a, b), k


def test_two_graphs_do_not_share_a_workspace():
    import gsr_train as G
    w = [torch.exp(torch.randn(100_000, generator=gen(k))).to(DEV) for k in (1, 2)]
    want = [G.keep_heaviest(x, 30_000) for x in w]
    graphs, outs = [], []
    for x in w:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(G.keep_heaviest(x, 30_000))
        graphs.append(g)
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for g, st in zip(graphs, s):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("through_a_view", [False, True])
def test_capture_is_refused_while_an_eager_graph_of_the_leaves_lives(through_a_view):
    """The accumulator of a leaf keeps the stream it was made on for as long as a graph of the leaf lives; a captured
    backward pass must not reach it.  Without that graph the capture works."""
    import gsr_train as G
    xyz, f, cam, up = scene(300, 4, 1, 5)
    x, fg = xyz.to(DEV).requires_grad_(), f.to(DEV).requires_grad_()
    cam, up = cam.to(DEV), up.to(DEV)
    q = G.mx4_quantize(fg.detach().flatten(1)[:, 3:])

    def trained():
        return G.sh_colors_quantized(x[:] if through_a_view else x, fg, cam, 1)

    def shown():
        return G.sh_colors(x[:] if through_a_view else x, fg.detach()[:, 0], q, cam, 1)

    for call in (trained, shown):
        eager = call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager graph of the same tensors"):
            with torch.cuda.graph(graph):
                call()
        with torch.cuda.graph(torch.cuda.CUDAGraph()):  # without gradients nothing is in the way
            with torch.no_grad():
                call()
        (want,) = torch.autograd.grad(eager, (x,), up)
        del eager
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            (got,) = torch.autograd.grad(call(), (x,), up)
        for _ in range(3):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


def test_capture_with_gradients_needs_the_compiled_binding(monkeypatch):
    import gsr_train as G
    from gsr_train import compact as T
    xyz, f, cam, _ = scene(40, 4, 1, 6)
    x, fg, cam = xyz.to(DEV).requires_grad_(), f.to(DEV), cam.to(DEV)
    monkeypatch.setattr(T, "_HOST", None)
    with pytest.raises(RuntimeError, match="gsr_host"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            G.sh_colors_quantized(x, fg, cam, 1)
