"""The drop-in rasterizer under torch.jit.trace: the traced module renders its inputs."""
import pytest
import torch

import harness as Hn
from gsr_tools.scene import orbit_camera, synthetic_scene

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("grad", [False, True])
def test_traced_rasterizer_renders(grad):
    from diff_gaussian_rasterization import GaussianRasterizer
    a, b = (synthetic_scene(2000, sh_degree=2, seed=s) for s in (5, 6))
    cam = orbit_camera(1, 160, 120, 150.0)
    rasterizer = GaussianRasterizer(Hn.settings_for(cam, 2, DEV))

    def fn(means, shs, opac, segs, scales, rots):
        color, radii, depth, alpha, segment = rasterizer(
            means3D=means, means2D=torch.zeros_like(means), opacities=opac, shs=shs, segments=segs, scales=scales,
            rotations=rots)
        return color, radii, depth, alpha, segment

    def inputs(s):
        t = (s.means3D, s.shs, s.opacities, s.segments, s.scales, s.rotations)
        return [x.to(DEV).contiguous().clone().requires_grad_(grad) for x in t]

    traced = torch.jit.trace(fn, tuple(inputs(a)), check_trace=False)
    args = inputs(b)
    got, want = traced(*args), fn(*args)
    assert float(want[0].detach().abs().sum()) > 0
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    if grad:
        up = torch.randn(want[0].shape, generator=torch.Generator().manual_seed(1)).to(DEV)
        for x, y in zip(torch.autograd.grad(got[0], args, up, allow_unused=True),
                        torch.autograd.grad(want[0], args, up, allow_unused=True)):
            assert (x is None) == (y is None) and (x is None or torch.equal(x, y))
