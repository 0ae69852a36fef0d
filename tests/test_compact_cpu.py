"""Compact-scene operators without a GPU: the C ABI, the refusals of both layers (before any
launch), and the oracle against cases worked out by hand."""
import ctypes
import os

import numpy as np
import pytest
import torch

from oracle import compact_oracle as O
from test_abi import declared_symbols

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_exports_every_compact_symbol():
    from diff_gaussian_rasterization import _C
    from gsr_train import compact as T
    syms = declared_symbols(os.path.join(ROOT, "include", "gsr_compact.h"))
    assert sorted(T.EXPORTED_SYMBOLS) == syms
    lib = ctypes.CDLL(_C.LIB_PATH)
    for s in syms:
        assert hasattr(lib, s)


def test_c_calls_validate_without_the_device():
    from gsr_train import compact as T
    L = T._lib
    err = lambda: L.gsr_last_error().decode()  # noqa: E731
    assert L.gsr_mx4_quantize(3, 45, None, 45, 16, 16, None) != 0 and "null buffer" in err()
    assert L.gsr_mx4_quantize(3, 45, 16, 44, 16, 16, None) != 0 and "overlap" in err()
    assert L.gsr_mx4_quantize(-1, 45, 16, 45, 16, 16, None) != 0
    assert L.gsr_mx4_quantize(0, 45, None, 45, None, None, None) == 0
    assert L.gsr_mx4_quantize(5, 0, None, 0, None, None, None) == 0
    assert L.gsr_mx4_dequantize(3, 45, 16, None, 16, None) != 0 and "null buffer" in err()
    assert L.gsr_sh_colors(0, 1, 3, 16, None, None, 3, None, None, None, None, None, None) == 0
    for V, deg, M in ((0, 0, 1), (17, 0, 1), (1, 4, 25), (1, 3, 15), (1, -1, 1), (1, 0, 17)):
        assert L.gsr_sh_colors(4, V, deg, M, 16, 16, 3, 16, 16, 16, 16, None, None) != 0
    assert L.gsr_sh_colors(4, 1, 1, 4, 16, 16, 3, None, 16, 16, 16, None, None) != 0 and "null buffer" in err()
    assert L.gsr_sh_colors_backward(4, 1, 1, 4, 16, 16, 16, 16, 16, None, 16, None, None, None) != 0
    assert L.gsr_sh_colors_backward(4, 1, 1, 4, 16, 16, 16, 16, None, 16, 16, None, None, None) != 0 and "null" in err()
    assert L.gsr_sh_colors_quantize(4, 1, 1, 4, 16, 16, 16, 16, 16, None, 16, None) != 0 and "null buffer" in err()
    assert L.gsr_sh_colors_backward(4, 1, 1, 4, 16, 16, 16, 16, None, None, None, None, None, None) == 0
    assert L.gsr_accumulate_weights(4, None, 1, 1.0, 16, None) != 0

    def groups(*g):
        return (T._Group * len(g))(*g)

    for bad in (groups((0, 5, 6, 0)), groups((0, 5, 2, 3)), groups((0, 11, 1, 0)), groups((3, 2, 0, 0)),
                groups((0, 5, 1, 0), (4, 8, 1, 0)), groups((0, 5, -1, 0))):
        assert L.gsr_keep_heaviest(10, 16, len(bad), bad, 16, 16, None) != 0
    assert L.gsr_keep_heaviest(10, None, 1, groups((0, 5, 1, 0)), 16, 16, None) != 0 and "null buffer" in err()
    assert L.gsr_keep_heaviest(10, 16, 65, groups(*[(0, 0, 0, 0)] * 65), 16, 16, None) != 0 and "64 groups" in err()
    assert L.gsr_keep_heaviest(10, None, 1, groups((0, 5, 0, 0)), None, None, None) == 0  # nothing to keep
    assert L.gsr_take_rows(3, None, 1, (T._Rows * 1)((16, 16, 3, 5, 0)), None) != 0
    assert L.gsr_take_rows(3, 16, 1, (T._Rows * 1)((16, None, 3, 5, 0)), None) != 0 and "null buffer" in err()
    assert L.gsr_take_rows(3, 16, 1, (T._Rows * 1)((16, 16, -3, 5, 0)), None) != 0
    assert L.gsr_take_rows(0, None, 1, (T._Rows * 1)((16, None, 3, 5, 0)), None) == 0
    # what is written overlaps: the source, the ids, another source, another destination, by its padding alone
    a, b, c, d = 0x10000, 0x20000, 0x30000, 0x40000
    for bad in ([(a, a, 3, 5, 0)], [(a, a + 48, 3, 5, 0)], [(a, d, 3, 5, 0)], [(a, b, 3, 5, 0), (b + 32, c, 3, 5, 0)],
                [(a, c, 3, 5, 0), (b, c + 32, 3, 5, 0)], [(a, b - 36, 3, 5, 1), (b, c, 3, 5, 0)]):
        assert L.gsr_take_rows(3, d, len(bad), (T._Rows * len(bad))(*bad), None) != 0 and "overlaps" in err()
    big = 2 ** 31 - 1
    assert L.gsr_sh_colors(big, 1, 0, 1, 16, 16, 3, None, None, 16, 16, None, None) != 0
    assert L.gsr_accumulate_weights(big, 16, 1, 1.0, 16, None) != 0


def refused(fn, *a, match, **k):
    with pytest.raises(RuntimeError, match=match):
        fn(*a, **k)


@pytest.mark.parametrize("route", ["host", "ctypes"])
def test_python_refusals(route, monkeypatch):
    """Both host routes, each with its own checks and the same messages."""
    import gsr_train as G
    from gsr_train import compact as T
    if route == "host" and T._HOST is None:
        pytest.skip("gsr_host not built from these sources (__graft_entry__.build())")
    if route == "ctypes":
        monkeypatch.setattr(T, "_HOST", None)
    z = torch.zeros
    refused(G.mx4_quantize, z(4, 45), match="GPU")
    refused(G.mx4_quantize, z(4, 45, dtype=torch.float16), match="float32")
    refused(G.mx4_quantize, [1.0], match="float32")
    refused(G.mx4_quantize, z(4, 15, 3), match="shape")
    u8 = torch.uint8
    codes, scales = z(5, 24, dtype=u8), z(5, 2, dtype=u8)
    rest = G.MX4Rows(codes, scales, 45)
    assert rest.rows == 5 and rest.nbytes == 5 * 26
    refused(G.MX4Rows, codes, scales, 44, match="codes|scales") if (44 + 7) // 8 * 4 != 24 else None
    refused(G.MX4Rows, codes, scales, 49, match="codes")
    refused(G.MX4Rows, codes, scales, -1, match="negative")
    refused(G.MX4Rows, codes.int(), scales, 45, match="uint8")
    refused(G.MX4Rows, codes, scales[:4], 45, match="rows")
    refused(G.MX4Rows, z(24, 5, dtype=u8).T, scales, 45, match="contiguous")
    refused(G.MX4Rows, z(5 * 24 + 1, dtype=u8)[1:].view(5, 24), scales, 45, match="multiple of 4")
    refused(rest.dequantize, match="GPU")
    xyz, dc, cam = z(5, 3), z(5, 1, 3), z(3)
    refused(G.sh_colors, xyz, dc, rest, cam, 3, match="GPU")
    refused(G.sh_colors, xyz, dc, rest, cam, 4, match="degree")
    refused(G.sh_colors, xyz, dc, rest, cam, 1.5, match="degree")
    refused(G.sh_colors, xyz, dc, rest, z(17, 3), 3, match="campos")
    refused(G.sh_colors, xyz, dc, rest, z(0, 3), 3, match="campos")
    refused(G.sh_colors, xyz, dc, rest, z(1, 4), 3, match="campos")
    refused(G.sh_colors, xyz, dc, codes, cam, 3, match="MX4Rows")
    refused(G.sh_colors, z(4, 3), z(4, 1, 3), rest, cam, 3, match="rows")
    refused(G.sh_colors, xyz, z(5, 2, 3), rest, cam, 3, match="features_dc")
    refused(G.sh_colors, xyz.double(), dc, rest, cam, 3, match="float32")
    refused(G.sh_colors, z(5, 2), dc, rest, cam, 3, match="xyz")
    small = G.MX4Rows(z(5, 8, dtype=u8), z(5, 1, dtype=u8), 9)
    refused(G.sh_colors, xyz, dc, small, cam, 2, match="degree")
    refused(G.sh_colors_quantized, xyz, z(5, 16, 3), cam, 3, match="GPU")
    refused(G.sh_colors_quantized, xyz, z(5, 17, 3), cam, 3, match="shape")
    refused(G.sh_colors_quantized, xyz, z(6, 16, 3), cam, 3, match="rows")
    refused(G.sh_colors_quantized, xyz, z(5, 9, 3), cam, 3, match="degree")
    w = z(10)
    refused(G.keep_heaviest, w, 5, match="GPU")
    refused(G.keep_heaviest, w, -1, match="negative")
    refused(G.keep_heaviest, w, 1, recent=-1, match="negative")
    refused(G.keep_heaviest, w, [1, 2], match="one budget")
    refused(G.keep_heaviest, w, 1, [(0, 4), (3, 8)], match="overlap")
    refused(G.keep_heaviest, w, 1, [(4, 8), (0, 3)], match="ascending")
    refused(G.keep_heaviest, w, 1, [(0, 11)], match="rows")
    refused(G.keep_heaviest, w, 1, [(0, 0)] * 65, match="64 groups")
    refused(G.keep_heaviest, w.int(), 1, match="float32")
    ids = z(2, dtype=torch.int32)
    refused(G.take_rows, ids, [z(4, 3)], match="GPU")
    refused(G.take_rows, ids.long(), [z(4, 3)], match="int32")
    refused(G.take_rows, ids, [z(4, 3).double()], match="float32 or int32")
    refused(G.take_rows, ids, [z(4, 6)[:, ::2]], match="contiguous")
    refused(G.take_rows, ids, [z(4, 3)], out=[z(3, 3)], match="out")
    refused(G.take_rows, ids, [z(4, 3)], out=[], match="one output")
    refused(G.accumulate_weights, w, z(9), match="shape")
    refused(G.accumulate_weights, w, w, match="GPU")


def test_feature_bits_are_4_or_32():
    from gsr_train import GaussianModel
    m = GaussianModel(1, device="cpu")
    assert m.feature_bits == 32
    m.feature_bits = 4
    with pytest.raises(ValueError, match="4 or 32"):
        m.feature_bits = 8


def test_keep_groups_cut_to_what_a_group_holds():
    from gsr_train.compact import _keep_groups
    assert _keep_groups("x", 10, 4, None, 0) == [(0, 10, 4, 0)]
    assert _keep_groups("x", 10, 40, None, 20) == [(0, 10, 10, 10)]
    assert _keep_groups("x", 10, [3, 9], [(0, 6), (6, 10)], [5, 1]) == [(0, 6, 3, 3), (6, 10, 4, 1)]
    assert _keep_groups("x", 0, 5, None, 1) == [(0, 0, 0, 0)]
    assert _keep_groups("x", 5, 5, [], 1) == []


def test_oracle_codes_by_hand():
    # largest 6: scale 1; every magnitude and every tie
    x = np.array([[6, 5, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, -6, -0.26, 0.24, 0, -0.0, 4.99, 5.01, 0.5]], np.float32)
    codes, scales = O.mx4_quantize(x)
    assert scales.tolist() == [[127]]
    want = [6, 4, 4, 2, 2, 1, 1, 0, -6, -0.5, 0, 0, 0, 4, 6, 0.5]
    assert O.mx4_dequantize(codes, scales, 16)[0].tolist() == want
    # the largest decides the power of two: 7.9 saturates, 8 doubles the scale
    for top, s, back in ((7.9, 127, 6.0), (8.0, 128, 8.0), (1e-45, 0, 0.0), (3.4e38, 252, 6 * 2.0 ** 125), (0.0, 0, 0.0)):
        codes, scales = O.mx4_quantize(np.array([[top]], np.float32))
        assert scales[0, 0] == s and O.mx4_dequantize(codes, scales, 1)[0, 0] == np.float32(back)
    # blocks do not share a scale; a NaN takes its block only
    x = np.zeros((1, 40), np.float32)
    x[0, 3], x[0, 35] = np.nan, 1.0
    d = O.mx4_dequantize(*O.mx4_quantize(x), 40)
    assert np.isnan(d[0, :32]).all() and d[0, 35] == 1.0 and (d[0, 36:] == 0).all()


def test_oracle_keep_by_hand():
    w = [5, 1, float("nan"), 5, 0, -0.0, float("inf"), 2, 9, 9]
    assert O.keep_heaviest(w, [(0, 10, 4, 0)]).tolist() == [0, 6, 8, 9]
    assert O.keep_heaviest(w, [(0, 10, 4, 3)]).tolist() == [6, 7, 8, 9]
    assert O.keep_heaviest(w, [(2, 6, 3, 0), (6, 8, 1, 1)]).tolist() == [3, 4, 5, 7]
    assert O.keep_heaviest([float("nan"), -float("inf"), -1], [(0, 3, 2, 0)]).tolist() == [1, 2]


@pytest.mark.parametrize("degree", [0, 1, 2, 3])
def test_oracle_basis_is_orthonormal(degree):
    """Integrals of products over the sphere (a product Gauss rule, exact at these degrees)."""
    t, wt = np.polynomial.legendre.leggauss(8)
    phi = np.arange(16) * (2 * np.pi / 16)
    z, p = np.meshgrid(t, phi, indexing="ij")
    r = np.sqrt(1 - z * z)
    d = torch.tensor(np.stack([r * np.cos(p), r * np.sin(p), z], -1).reshape(-1, 3))
    w = torch.tensor((wt[:, None] * np.full(16, 2 * np.pi / 16)).reshape(-1))
    b = O.sh_values(d, degree)
    # the constants are written with 16 digits or less: 1e-12
    assert torch.allclose((b * w[:, None]).T @ b, torch.eye(b.shape[1], dtype=torch.float64), atol=1e-12)


def test_take_rows_of_nothing_overlaps_nothing():
    """An empty destination or source inside another tensor's range is no clash."""
    from gsr_train import compact as T
    table = (T._Rows * 2)((4096, 4160, 4, 0, 0), (4096, 4104, 0, 64, 0))
    assert T._lib.gsr_take_rows(0, 64, 2, table, None) == 0
    table = (T._Rows * 1)((4100, 4096, 2, 0, 0))
    assert T._lib.gsr_take_rows(0, 64, 1, table, None) == 0


def _contribution_worker(rank, world, port, out_q):
    import sys
    sys.path[:0] = [ROOT, os.path.join(ROOT, "3d_gaussian_magic_change-segment_3dgs_amd")]
    import torch.distributed as dist
    from gsr_tools import dp
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world)
    weights = torch.rand(100, 1, generator=torch.Generator().manual_seed(rank))
    dp.reduce_contribution(weights)
    out_q.put((rank, weights.numpy().copy()))
    dist.barrier()
    dist.destroy_process_group()


def test_contribution_reduction_gloo_ws2():
    """Every rank gets the same sums, bit for bit: what evict() keeps is the same everywhere."""
    import torch.multiprocessing as mp
    from test_dist_cpu import _free_port
    ctx = mp.get_context("spawn")
    q, port = ctx.Queue(), _free_port()
    procs = [ctx.Process(target=_contribution_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = dict(q.get(timeout=120) for _ in range(2))
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    a, b = (torch.rand(100, 1, generator=torch.Generator().manual_seed(r)).numpy() for r in range(2))
    assert np.array_equal(res[0], a + b) and np.array_equal(res[1], res[0])
