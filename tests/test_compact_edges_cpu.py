"""Compact-scene operators without a GPU: arguments at the edges of what a call takes (tests/test_compact_cpu.py has
the ordinary refusals)."""
import pytest
import torch

from test_compact_cpu import refused


@pytest.fixture(params=["host", "ctypes"])
def route(request, monkeypatch):
    """Both host routes."""
    from gsr_train import compact as T
    if request.param == "host" and T._HOST is None:
        pytest.skip("gsr_host not built from these sources (__graft_entry__.build())")
    if request.param == "ctypes":
        monkeypatch.setattr(T, "_HOST", None)
    return request.param


def test_sizes_that_do_not_fit_an_int_are_refused(route):
    """Tensors without memory: what counts is that no size is cut to 32 bits on its way to the library."""
    import gsr_train as G
    meta = lambda *s, **k: torch.empty(*s, device="meta", **k)  # noqa: E731
    for n in (2 ** 31, 2 ** 32 + 7):
        refused(G.accumulate_weights, meta(n), meta(n), match="2\\^31")
        refused(G.keep_heaviest, meta(n), 5, match="2\\^31")
    for K in (2 ** 20 + 1, 2 ** 31, 2 ** 32 + 45):
        refused(G.mx4_quantize, meta(1, K), match="2\\^20")
        words, blocks = (K + 7) // 8, (K + 31) // 32
        rows = G.MX4Rows(meta(1, 4 * words, dtype=torch.uint8), meta(1, blocks, dtype=torch.uint8), K)
        refused(rows.dequantize, match="2\\^20")
    refused(G.mx4_quantize, meta(3, 2 ** 20), match="GPU")  # the widest
    refused(G.mx4_quantize, meta(0, 2 ** 21), match="GPU")  # nothing of any width


def test_budgets_are_whole_numbers(route):
    """A share of the rows is no budget: it would be cut to 0, and everything would go."""
    import gsr_train as G
    from gsr_train.compact import _keep_groups
    w = torch.zeros(10)
    for bad in (0.7, 2.5, [3, 0.5], float("nan"), float("inf"), torch.tensor(0.5), None, "5"):
        refused(G.keep_heaviest, w, bad, [(0, 4), (4, 10)], match="whole numbers")
        refused(G.keep_heaviest, w, 1, [(0, 4), (4, 10)], recent=bad, match="whole numbers")
    refused(G.keep_heaviest, w, 1, [(0, 4.5)], match="whole numbers")
    assert _keep_groups("x", 10, 1e1, [(0, 6.0), (torch.tensor(6), 10)], torch.tensor(2)) == [(0, 6, 6, 2), (6, 10, 4, 2)]


def test_accumulated_weights_that_overlap_their_sum_are_refused():
    """acc and weights in the same memory: only element on element (acc <- (decay + 1) acc) has one result."""
    from gsr_train import compact as T
    L = T._lib
    call = lambda P, w, stride, acc: (L.gsr_accumulate_weights(P, w, stride, 1.0, acc, None),  # noqa: E731
                                      L.gsr_last_error().decode())
    a = 1 << 20
    for P, w, stride in ((10, a + 4, 1), (10, a - 4, 1), (10, a - 36, 1), (10, a + 36, 1), (10, a, 2), (10, a - 8, 4),
                         (10, a, 0), (10, a + 16, 0), (10, a - 36, 3), (2, a - 4, 1), (10, a + 36, -1), (10, a + 76, -2)):
        rc, err = call(P, w, stride, a)
        assert rc != 0 and "overlap" in err, (P, w - a, stride)


def test_calls_larger_than_a_grid_are_refused_by_name():
    """A launch has fewer than 2^32 threads: 2^24 - 1 blocks of 256."""
    from gsr_train import compact as T
    L = T._lib
    err = lambda: L.gsr_last_error().decode()  # noqa: E731
    most = 2 ** 24 - 1
    for R, K in ((most * 1024 // 45 + 1, 45), (most * 1024 // 4 + 1, 4), (most * 256 + 1, 1), (most * 128 + 1, 34),
                 (most + 1, 1024), (most // 2, 4096)):  # 1024 values a block, or 256 pieces of four
        assert L.gsr_mx4_dequantize(R, K, 4096, 4096, 4096, None) != 0 and "too many rows in one call" in err(), (R, K)
    for R, K in ((most * 128 + 1, 9), (most * 64 + 1, 45), (most + 1, 32 * 128), (most, 32 * 129)):  # 128 blocks of 32
        assert L.gsr_mx4_quantize(R, K, 4096, K, 4096, 4096, None) != 0 and "too many rows in one call" in err(), (R, K)


# ---- the counters of the benchmark line -----------------------------------------------------------
def test_counters_stand_for_the_sources_of_the_kernels_they_describe(tmp_path, monkeypatch):
    """The committed counter summary is the renderer's: it holds as long as the renderer's sources stay, whatever
    other sources the library is linked from."""
    import os
    import shutil
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    monkeypatch.syspath_prepend(root)
    monkeypatch.syspath_prepend(os.path.join(root, "tools"))
    import bench
    import pmc_summary
    summary, note = bench.pmc_for_this_build()
    assert summary is not None, note
    bwd = summary["kernels"]["render_bwd"]
    assert bwd["hbm_bytes_per_launch"] > 0 and bwd["SQ_INSTS_VALU"] > 0
    pkg = "3d_gaussian_magic_change-segment_3dgs_amd"
    shutil.copytree(os.path.join(root, pkg, "csrc"), tmp_path / pkg / "csrc")
    shutil.copytree(os.path.join(root, "include"), tmp_path / "include")
    monkeypatch.setattr(pmc_summary, "ROOT", str(tmp_path))
    csrc = tmp_path / pkg / "csrc"
    assert pmc_summary.sources_sha256() == summary["sources_sha256"]
    (csrc / "compact.hip").write_text("// other kernels\n")
    assert pmc_summary.sources_sha256() == summary["sources_sha256"]
    for name in ("render_bwd.hip", "api.hip", "gsr_internal.h", "new.hip"):
        old = (csrc / name).read_text() if (csrc / name).exists() else None
        (csrc / name).write_text((old or "") + "\n")
        assert pmc_summary.sources_sha256() != summary["sources_sha256"], name
        if old is None:
            (csrc / name).unlink()
        else:
            (csrc / name).write_text(old)
    assert "pmc_summary" in sys.modules


def test_rows_of_codes_fit_every_width_of_their_words():
    """24 bytes of codes and 2 scales are rows of 41 to 48 values."""
    import gsr_train as G
    codes, scales = torch.zeros(5, 24, dtype=torch.uint8), torch.zeros(5, 2, dtype=torch.uint8)
    for width in range(41, 49):
        assert G.MX4Rows(codes, scales, width).width == width
    refused(G.MX4Rows, codes, scales, 40, match="codes")
    refused(G.MX4Rows, codes, scales, 49, match="codes")
    refused(G.MX4Rows, codes, scales[:, :1].contiguous(), 44, match="scales")
