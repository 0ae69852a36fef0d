"""Definitions of the compact-scene operators (include/gsr_compact.h) in numpy / torch on
the CPU, in 64 bits: the test oracle of tests/test_gpu_compact.py."""
import numpy as np
import torch

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def mx4_quantize(x):
    """float32 rows [R, K] -> (codes uint8 [R, 4 ceil(K/8)], scales uint8 [R, ceil(K/32)])."""
    x = np.asarray(x, dtype=np.float32)
    R, K = x.shape
    nb, nw = -(-K // 32), -(-K // 8)
    code = np.zeros((R, 8 * nw), dtype=np.uint8)
    scales = np.zeros((R, nb), dtype=np.uint8)
    for r in range(R):
        for b in range(nb):
            blk = x[r, 32 * b:32 * b + 32].astype(np.float64)
            if not np.isfinite(blk).all():
                scales[r, b] = 255
                continue
            top = np.abs(blk).max()
            e = -127 if top == 0 else max(int(np.frexp(top)[1]) - 1 - 2, -127)
            scales[r, b] = e + 127
            y = np.abs(np.ldexp(blk, -e))
            d = np.abs(y[:, None] - MAGNITUDES[None, :])
            for k in range(len(blk)):  # nearest, of two equally near ones the even index
                near = np.flatnonzero(d[k] == d[k].min())
                best = near[near % 2 == 0][0] if len(near) > 1 else near[0]
                code[r, 32 * b + k] = best + 8 * np.signbit(blk[k])
    return (code[:, 0::2] | code[:, 1::2] << 4), scales


def mx4_dequantize(codes, scales, K):
    """-> float32 [R, K]."""
    codes, scales = np.asarray(codes), np.asarray(scales)
    R = codes.shape[0]
    nib = np.empty((R, 2 * codes.shape[1]), dtype=np.int64)
    nib[:, 0::2], nib[:, 1::2] = codes & 15, codes >> 4
    nib = nib[:, :K]
    s = np.repeat(scales.astype(np.int64), 32, axis=1)[:, :K]
    v = np.ldexp(MAGNITUDES[nib & 7], s - 127) * np.where(nib & 8, -1.0, 1.0)
    return np.where(s == 255, np.nan, v).astype(np.float32)


def sh_values(d, degree):
    """Real spherical harmonics [..., (degree+1)^2] of unit vectors d (utils/sh_utils.py:57-112)."""
    x, y, z = d.unbind(-1)
    b = [torch.full_like(x, 0.28209479177387814)]
    if degree > 0:
        b += [-0.4886025119029199 * y, 0.4886025119029199 * z, -0.4886025119029199 * x]
    if degree > 1:
        b += [1.0925484305920792 * x * y, -1.0925484305920792 * y * z,
              0.31539156525252005 * (2 * z * z - x * x - y * y), -1.0925484305920792 * x * z,
              0.5462742152960396 * (x * x - y * y)]
    if degree > 2:
        b += [-0.5900435899266435 * y * (3 * x * x - y * y), 2.890611442640554 * x * y * z,
              -0.4570457994644658 * y * (4 * z * z - x * x - y * y),
              0.3731763325901154 * z * (2 * z * z - 3 * x * x - 3 * y * y),
              -0.4570457994644658 * x * (4 * z * z - x * x - y * y), 1.445305721320277 * z * (x * x - y * y),
              -0.5900435899266435 * x * (x * x - 3 * y * y)]
    return torch.stack(b, -1)


def sh_preclamp(xyz, coef, campos, degree):
    """float64 values before the clamp [V, P, 3]; coef [P, M, 3] (decoded)."""
    u = xyz.double()[None] - campos.double()[:, None]
    n = u.norm(dim=2, keepdim=True)
    d = torch.where(n > 0, u / torch.where(n > 0, n, torch.ones_like(n)), torch.zeros_like(u))
    b = sh_values(d, degree)
    return 0.5 + torch.einsum("vpk,pkc->vpc", b, coef.double()[:, :b.shape[-1]])


def keep_heaviest(weights, plan):
    """plan: [(begin, end, keep, recent)] -> ids int32."""
    w = np.asarray(weights, dtype=np.float32).astype(np.float64)
    rank = np.where(np.isnan(w), -np.inf, w)
    out = []
    for a, b, keep, recent in plan:
        old = b - recent
        # heaviest first, NaN behind -inf, then the lowest row
        order = sorted(range(a, old), key=lambda i: (-rank[i], bool(np.isnan(w[i])), i))
        out += sorted(order[:keep - recent]) + list(range(old, b))
    return np.array(out, dtype=np.int32)
