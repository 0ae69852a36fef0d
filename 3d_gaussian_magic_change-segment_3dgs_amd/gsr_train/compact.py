"""Compact scenes: fewer Gaussians, fewer bytes each (kernels: include/gsr_compact.h,
csrc/compact.hip).

* `mx4_quantize` / `MX4Rows`: rows of floats -- the SH coefficients above the constant
  one, 180 of a Gaussian's 244 bytes -- in 4-bit microscaled floating point (26 bytes).
* `sh_colors`: view-dependent colours straight from the codes, with gradients for the
  positions and the constant coefficients; `sh_colors_quantized`: the same from the fp32
  features, which are rounded to 4 bits in the call and get their gradient straight
  through the rounding (training a scene that will be stored in 4 bits).  Both stand where
  the reference evaluates SH in Python (gaussian_renderer/__init__.py:349-357,
  convert_SHs_python) and go to the rasterizer as colors_precomp.
* `keep_heaviest` / `take_rows`: a scene, or each scene of a merged model, brought to a
  budget of Gaussians by accumulated blend weight.
* `CompactGaussians`: a trained model with the coefficients in 4 bits, for rendering.

All tensors are float32 (ids int32, codes and scales uint8) on one GPU; a call uses that
GPU's current stream, takes its workspace from torch's allocator and never waits for the
device, so it can be captured into a graph.  A pass with gradients is captured forward and
backward together, with no eager graph of the same leaves alive: that is refused, since the
captured backward pass would have to wait on the eager graph's stream.  torch.jit.trace records
sh_colors and sh_colors_quantized as calls of them; the other operators, and all of them under
make_fx, refuse to be traced."""
import ctypes
import numbers

import torch
from torch.fx.experimental.proxy_tensor import get_proxy_mode

from . import _C
from diff_gaussian_rasterization._C import MAX_VIEWS, _HOST

_lib = _C._lib
_vp, _i, _ll, _f = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float

MX_BLOCK = 32    # include/gsr_compact.h GSR_MX_BLOCK
MAX_WIDTH = 1 << 20  # GSR_MAX_WIDTH
MAX_GROUPS = 64  # GSR_KEEP_MAX_GROUPS


class _Group(ctypes.Structure):
    _fields_ = [("begin", _i), ("end", _i), ("keep", _i), ("recent", _i)]


class _Rows(ctypes.Structure):
    _fields_ = [("src", _vp), ("dst", _vp), ("width", _i), ("rows", _i), ("pad", _i)]


for _name, _args in (("gsr_mx4_quantize", [_ll, _i, _vp, _ll, _vp, _vp, _vp]),
                     ("gsr_mx4_dequantize", [_ll, _i, _vp, _vp, _vp, _vp]),
                     ("gsr_sh_colors", [_i, _i, _i, _i, _vp, _vp, _ll, _vp, _vp, _vp, _vp, _vp, _vp]),
                     ("gsr_sh_colors_quantize", [_i, _i, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp]),
                     ("gsr_sh_colors_backward", [_i, _i, _i, _i] + [_vp] * 10),
                     ("gsr_accumulate_weights", [_i, _vp, _ll, _f, _vp, _vp]),
                     ("gsr_keep_heaviest", [_i, _vp, _i, ctypes.POINTER(_Group), _vp, _vp, _vp]),
                     ("gsr_take_rows", [_i, _vp, _i, ctypes.POINTER(_Rows), _vp])):
    getattr(_lib, _name).restype = _i
    getattr(_lib, _name).argtypes = _args
_lib.gsr_keep_ws_bytes.restype = ctypes.c_size_t
_lib.gsr_keep_ws_bytes.argtypes = [_i]

EXPORTED_SYMBOLS = ("gsr_mx4_quantize", "gsr_mx4_dequantize", "gsr_sh_colors", "gsr_sh_colors_quantize",
                    "gsr_sh_colors_backward",
                    "gsr_accumulate_weights", "gsr_keep_ws_bytes", "gsr_keep_heaviest", "gsr_take_rows")


def _typed(what, dtype=torch.float32, **tensors):
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor) or t.dtype != dtype:
            raise RuntimeError(f"{what}: {name} must be a {dtype} tensor (got "
                               f"{t.dtype if isinstance(t, torch.Tensor) else type(t).__name__})")


def _on_gpu(what, first, **others):
    """`first` is a GPU tensor and the others are on its device."""
    if first.device.type != "cuda":
        raise RuntimeError(f"{what}: tensors must be on the GPU (the HIP path has no CPU fallback)")
    for name, t in others.items():
        if t.device != first.device:
            raise RuntimeError(f"{what}: {name} is on {t.device}, expected {first.device}")


def _trace_check(what, jit=True):
    """A tracer would record the allocations and not the kernels: what it made would return uninitialised memory."""
    if (jit and torch._C._get_tracing_state() is not None) or get_proxy_mode() is not None:
        raise RuntimeError(f"{what}: cannot be traced")


def _call(device, fn, *args):
    """fn on `device` and its current stream."""
    with torch.cuda.device(device):
        _C._check(fn(*args, _C._stream(device)))


def _written(t):
    """Tells autograd of a write through the pointer."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _width_check(what, K):
    if K > MAX_WIDTH:  # (the library takes a width as an int)
        raise RuntimeError(f"{what}: rows of more than 2^20 values")


def _words(K):
    return (K + 7) // 8


def _blocks(K):
    return (K + MX_BLOCK - 1) // MX_BLOCK


# ---- 4-bit rows ------------------------------------------------------------------------
class MX4Rows:
    """R rows of `width` floats in 4-bit microscaled floating point: `codes` uint8
    [R, 4 ceil(width / 8)] (two codes a byte, the earlier value in the low half, rows
    padded with zeros to 32-bit words), `scales` uint8 [R, ceil(width / 32)] (2^(byte - 127)
    for 32 neighbouring values of a row; 255: the block held a NaN or an infinity)."""

    def __init__(self, codes, scales, width):
        width = int(width)
        if width < 0:
            raise RuntimeError("MX4Rows: width must not be negative")
        for t, name, cols in ((codes, "codes", 4 * _words(width)), (scales, "scales", _blocks(width))):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8 or t.dim() != 2 or t.shape[1] != cols:
                raise RuntimeError(f"MX4Rows: {name} must be a uint8 tensor of shape (rows, {cols}) for width {width}")
            if not t.is_contiguous():
                raise RuntimeError(f"MX4Rows: {name} must be contiguous")
        if codes.shape[0] != scales.shape[0] or codes.device != scales.device:
            raise RuntimeError("MX4Rows: codes and scales must have the same rows and device")
        if codes.numel() and codes.data_ptr() % 4:
            raise RuntimeError("MX4Rows: codes must start at a multiple of 4 bytes")
        self.codes, self.scales, self.width = codes, scales, width

    rows = property(lambda self: self.codes.shape[0])
    device = property(lambda self: self.codes.device)
    nbytes = property(lambda self: self.codes.numel() + self.scales.numel())

    def dequantize(self):
        """The values the codes stand for, float32 [rows, width] (each is exact)."""
        if _HOST is not None:
            return _HOST.mx4_dequantize(self.codes, self.scales, self.width)
        _trace_check("MX4Rows.dequantize")
        if self.rows:
            _width_check("MX4Rows.dequantize", self.width)
        _on_gpu("MX4Rows.dequantize", self.codes)
        x = torch.empty((self.rows, self.width), dtype=torch.float32, device=self.device)
        if x.numel():
            _call(self.device, _lib.gsr_mx4_dequantize, self.rows, self.width, self.codes.data_ptr(),
                  self.scales.data_ptr(), x.data_ptr())
        return x

    def to(self, device):
        return MX4Rows(self.codes.to(device), self.scales.to(device), self.width)


def _quantize(x2):
    """x2 [R, K] with contiguous values in a row -> (codes, scales)."""
    R, K = x2.shape
    codes = torch.empty((R, 4 * _words(K)), dtype=torch.uint8, device=x2.device)
    scales = torch.empty((R, _blocks(K)), dtype=torch.uint8, device=x2.device)
    if R and K:
        _call(x2.device, _lib.gsr_mx4_quantize, R, K, x2.data_ptr(), x2.stride(0), codes.data_ptr(), scales.data_ptr())
    return codes, scales


def mx4_quantize(x):
    """Rows of a float32 GPU tensor [R, K] -> MX4Rows (blocks of 32 neighbours of a row;
    the conversion is described in include/gsr_compact.h).  A view whose rows lie apart
    (features[:, 1:].flatten(1)) is read in place."""
    if _HOST is not None and isinstance(x, torch.Tensor):
        codes, scales = _HOST.mx4_quantize(x)
    else:
        _trace_check("mx4_quantize")
        _typed("mx4_quantize", x=x)
        if x.dim() != 2:
            raise RuntimeError("mx4_quantize: x must have shape (rows, values)")
        if x.shape[0]:
            _width_check("mx4_quantize", x.shape[1])
        _on_gpu("mx4_quantize", x)
        if x.numel() and ((x.shape[1] > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < x.shape[1])):
            x = x.contiguous()
        codes, scales = _quantize(x)
    q = MX4Rows.__new__(MX4Rows)  # (nothing to check)
    q.codes, q.scales = codes, scales
    q.width = x.shape[1]
    return q


# ---- colours -----------------------------------------------------------------------------
def _sh_check(what, xyz, campos, degree, M):
    _typed(what, xyz=xyz, campos=campos)
    if xyz.dim() != 2 or xyz.shape[1] != 3 or xyz.shape[0] >= 2 ** 31:
        raise RuntimeError(f"{what}: xyz must have shape (P, 3), P below 2^31")
    if campos.shape != (3,) and (campos.dim() != 2 or campos.shape[1] != 3 or not 1 <= campos.shape[0] <= MAX_VIEWS):
        raise RuntimeError(f"{what}: campos must have shape (3,) or (V, 3) with V of 1..{MAX_VIEWS}")
    if int(degree) != degree or not 0 <= degree <= 3 or (degree + 1) ** 2 > M:
        raise RuntimeError(f"{what}: degree must be 0..3 and the features must hold its coefficients "
                           f"(degree {degree}, {M} coefficients)")


def _forward_check(what, *tensors):
    if any(torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what}: there is no forward-mode derivative")


def _capture_check(what, *tensors):
    """The compiled binding looks for eager graphs of the same tensors, whose streams a captured backward pass
    must not touch; here there is no way to."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors) and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what}: capturing a pass with gradients needs the compiled host binding (gsr_host)")


def _buffers(xyz, V, single, grad):
    """(colors [V, P, 3] or [P, 3], mask [V, P] for the backward or None)."""
    P, dev = xyz.shape[0], xyz.device
    colors = torch.empty((P, 3) if single else (V, P, 3), dtype=torch.float32, device=dev)
    return colors, torch.empty((V, P), dtype=torch.uint8, device=dev) if grad else None


def _ptr(t):
    return None if t is None else t.data_ptr()


class _NoSecondDerivative(torch.autograd.Function):
    """A gradient as a function of `of`, whose derivative is refused."""

    @staticmethod
    def forward(ctx, gradient, *of):
        return gradient.clone()

    @staticmethod
    def backward(ctx, g):
        raise RuntimeError("sh_colors: trying to differentiate twice (the colours are once_differentiable)")


def _once(gradient, *of):
    of = [t for t in of if t is not None and t.requires_grad]
    if gradient is None or not of or not torch.is_grad_enabled():
        return gradient
    return _NoSecondDerivative.apply(gradient, *of)


@torch.no_grad()
def _backward(g, saved, degree, M, dxyz, ddc, dfeatures):
    xyz, campos, codes, scales, mask = saved
    P = xyz.shape[0]
    if P:
        g = g.contiguous()
        _call(xyz.device, _lib.gsr_sh_colors_backward, P, campos.shape[0], degree, M, xyz.data_ptr(), codes.data_ptr(),
              scales.data_ptr(), campos.data_ptr(), mask.data_ptr(), g.data_ptr(), _ptr(dxyz), _ptr(ddc),
              _ptr(dfeatures))


class _ShColors(torch.autograd.Function):
    """colors [V, P, 3] ([P, 3] with `single`) from xyz, the constant coefficients dc [P, 3] and codes."""

    @staticmethod
    def forward(ctx, xyz, dc, campos, codes, scales, degree, M, single):
        P, V = xyz.shape[0], campos.shape[0]
        colors, mask = _buffers(xyz, V, single, any(ctx.needs_input_grad))
        if P:
            _call(xyz.device, _lib.gsr_sh_colors, P, V, degree, M, xyz.data_ptr(), dc.data_ptr(), dc.stride(0),
                  codes.data_ptr(), scales.data_ptr(), campos.data_ptr(), colors.data_ptr(), _ptr(mask))
        ctx.save_for_backward(xyz, campos, codes, scales, mask)
        ctx.degree, ctx.M = degree, M
        return colors

    @staticmethod
    def backward(ctx, g):
        xyz = ctx.saved_tensors[0]
        dxyz = torch.empty_like(xyz) if ctx.needs_input_grad[0] else None
        ddc = torch.empty_like(xyz) if ctx.needs_input_grad[1] else None
        _backward(g, ctx.saved_tensors, ctx.degree, ctx.M, dxyz, ddc, None)
        if ctx.degree > 0:
            dxyz = _once(dxyz, g, xyz)
        return dxyz, _once(ddc, g), None, None, None, None, None, None


class _ShColorsQuantized(torch.autograd.Function):
    """colors [V, P, 3] ([P, 3] with `single`) from xyz and fp32 features [P, M, 3]; what is kept
    of the features for the backward are their codes, 26 bytes a Gaussian, and a byte a view."""

    @staticmethod
    def forward(ctx, xyz, features, campos, degree, single, history):
        P, M = features.shape[:2]
        K, V, dev = 3 * (M - 1), campos.shape[0], xyz.device
        codes = torch.empty((P, 4 * _words(K)), dtype=torch.uint8, device=dev)
        scales = torch.empty((P, _blocks(K)), dtype=torch.uint8, device=dev)
        colors, mask = _buffers(xyz, V, single, True)
        if P:
            _call(dev, _lib.gsr_sh_colors_quantize, P, V, degree, M, xyz.data_ptr(), features.data_ptr(),
                  campos.data_ptr(), codes.data_ptr(), scales.data_ptr(), mask.data_ptr(), colors.data_ptr())
        ctx.save_for_backward(xyz, campos, codes, scales, mask)
        ctx.degree, ctx.M, ctx.history = degree, M, history
        return colors

    @staticmethod
    def backward(ctx, g):
        xyz = ctx.saved_tensors[0]
        dxyz = torch.empty_like(xyz) if ctx.needs_input_grad[0] else None
        df = None
        if ctx.needs_input_grad[1]:
            df = torch.empty((xyz.shape[0], ctx.M, 3), dtype=torch.float32, device=xyz.device)
        _backward(g, ctx.saved_tensors, ctx.degree, ctx.M, dxyz, None, df)
        if ctx.degree > 0:  # (straight through the rounding: df is no function of the features)
            return _once(dxyz, g, xyz, *ctx.history), _once(df, g, xyz), None, None, None, None
        return dxyz, _once(df, g), None, None, None, None


def _plain(a, b, c, degree):
    """What the C++ binding takes; anything else is refused (or converted) below."""
    return isinstance(a, torch.Tensor) and isinstance(b, torch.Tensor) and isinstance(c, torch.Tensor) and \
        (type(degree) is int or isinstance(degree, numbers.Integral))


def sh_colors(xyz, features_dc, rest, campos, degree):
    """max(0, 1/2 + sum_k Y_k(d) coefficient_k), d the direction from the camera to the
    Gaussian, for coefficients held in 4 bits (utils/sh_utils.py:57-112 and the + 0.5 and
    clamp of gaussian_renderer/__init__.py:354-355).

    xyz [P, 3], features_dc [P, 1, 3] or [P, 3], rest an MX4Rows of P rows of 3 (M - 1)
    values, campos [3] -> colors [P, 3], or [V, 3] -> [V, P, 3].  Differentiable in xyz and
    features_dc (gradients summed over the views; campos gets none, nor do the codes); a
    channel that the clamp holds at zero gives no gradient, and a Gaussian at the camera
    position itself none to xyz.  Second derivatives and forward mode are refused.  A
    features_dc of its own ([P, 3] contiguous) is read faster than a view of [P, M, 3] features,
    whose rows lie a cache line apart."""
    if _HOST is not None and isinstance(rest, MX4Rows) and _plain(xyz, features_dc, campos, degree):
        colors = _HOST.sh_colors(xyz, features_dc, rest.codes, rest.scales, rest.width, campos, degree)
        if colors is not None:  # (None under torch.jit.trace, which records the Python function below)
            return colors
    _trace_check("sh_colors", jit=False)
    if not isinstance(rest, MX4Rows) or rest.width % 3 or rest.width > 45:
        raise RuntimeError("sh_colors: rest must be MX4Rows of 3 (M - 1) values, M of 1..16")
    M = rest.width // 3 + 1
    _sh_check("sh_colors", xyz, campos, degree, M)
    P = xyz.shape[0]
    _typed("sh_colors", features_dc=features_dc)
    if features_dc.shape not in ((P, 1, 3), (P, 3)):
        raise RuntimeError(f"sh_colors: features_dc must have shape ({P}, 1, 3) or ({P}, 3)")
    if rest.rows != P:
        raise RuntimeError(f"sh_colors: rest must have {P} rows (got {rest.rows})")
    _on_gpu("sh_colors", xyz, features_dc=features_dc, rest=rest, campos=campos)
    _forward_check("sh_colors", xyz, features_dc, campos)
    _capture_check("sh_colors", xyz, features_dc)
    dc = features_dc.reshape(P, 3)
    if P and (dc.stride(1) != 1 or (P > 1 and dc.stride(0) < 3)):
        dc = dc.contiguous()
    return _ShColors.apply(xyz.contiguous(), dc, campos.detach().reshape(-1, 3).contiguous(), rest.codes, rest.scales,
                           int(degree), M, campos.dim() == 1)


def sh_colors_quantized(xyz, features, campos, degree):
    """sh_colors of features [P, M, 3] (fp32, coefficient 0 the constant one) whose
    coefficients above the constant one are rounded to 4 bits in the call: the colours a
    model shows after `compact()`.  Differentiable in xyz and features; the gradient goes
    straight through the rounding, and coefficients above `degree` get zero."""
    if _HOST is not None and _plain(xyz, features, campos, degree):
        colors = _HOST.sh_colors_quantized(xyz, features, campos, degree)
        if colors is not None:  # (as sh_colors)
            return colors
    what = "sh_colors_quantized"
    _trace_check(what, jit=False)
    _typed(what, features=features)
    if features.dim() != 3 or features.shape[2] != 3 or not 1 <= features.shape[1] <= 16:
        raise RuntimeError(f"{what}: features must have shape (P, M, 3), M of 1..16")
    _sh_check(what, xyz, campos, degree, features.shape[1])
    if features.shape[0] != xyz.shape[0]:
        raise RuntimeError(f"{what}: features must have {xyz.shape[0]} rows (got {features.shape[0]})")
    _on_gpu(what, xyz, features=features, campos=campos)
    _forward_check(what, xyz, features, campos)
    _capture_check(what, xyz, features)
    # (an empty tensor that comes from the features, not their memory: what a gradient of the positions depends on)
    history = (features[:0].clone(),) if torch.is_grad_enabled() and xyz.requires_grad else ()
    return _ShColorsQuantized.apply(xyz.contiguous(), features.contiguous(),
                                    campos.detach().reshape(-1, 3).contiguous(), int(degree), campos.dim() == 1, history)


# ---- eviction to a budget --------------------------------------------------------------------
@torch.no_grad()
def accumulate_weights(acc, weights, decay=1.0):
    """acc <- decay * acc + weights, in place: acc float32 contiguous of P values, weights
    float32 [P] of any stride (a column of a [P, 3] gradient), which may be acc itself but not
    overlap it otherwise."""
    if _HOST is not None and isinstance(acc, torch.Tensor) and isinstance(weights, torch.Tensor):
        return _HOST.accumulate_weights(acc, weights, float(decay))
    _trace_check("accumulate_weights")
    _typed("accumulate_weights", acc=acc, weights=weights)
    P = acc.numel()
    if P >= 2 ** 31:
        raise RuntimeError("accumulate_weights: at most 2^31 - 1 weights")
    if not acc.is_contiguous() or weights.dim() != 1 or weights.shape[0] != P:
        raise RuntimeError("accumulate_weights: acc must be contiguous and weights have shape (P,), P values each")
    _on_gpu("accumulate_weights", acc, weights=weights)
    if P:
        _call(acc.device, _lib.gsr_accumulate_weights, P, weights.data_ptr(), weights.stride(0), float(decay),
              acc.data_ptr())
        _written(acc)


def _whole(what, v):
    """v as an int (which int() alone would make of a share of the rows too: 0)."""
    if type(v) is int:
        return v
    try:
        n = int(v)
    except (TypeError, ValueError, OverflowError):
        n = None
    if n is None or n != v:
        raise RuntimeError(f"{what}: budgets, recent and groups must be whole numbers (got {v!r})")
    return n


def _keep_groups(what, P, budgets, groups, recent):
    """[(begin, end, keep, recent)] with keep and recent cut to what the group holds."""
    groups = [(0, P)] if groups is None else [(_whole(what, a), _whole(what, b)) for a, b in groups]
    each = lambda v: [_whole(what, x) for x in v] if isinstance(v, (list, tuple)) else \
        [_whole(what, v)] * len(groups)  # noqa: E731
    budgets, recent = each(budgets), each(recent)
    if len(budgets) != len(groups) or len(recent) != len(groups):
        raise RuntimeError(f"{what}: one budget (and one recent) for each of the {len(groups)} groups, or one for all")
    if len(groups) > MAX_GROUPS:
        raise RuntimeError(f"{what}: at most {MAX_GROUPS} groups a call (got {len(groups)})")
    last, out = 0, []
    for (a, b), k, r in zip(groups, budgets, recent):
        if not last <= a <= b <= P:
            raise RuntimeError(f"{what}: groups must be ascending (begin, end) ranges of the {P} rows, without overlap")
        if k < 0 or r < 0:
            raise RuntimeError(f"{what}: budget and recent must not be negative")
        last, k = b, min(k, b - a)
        out.append((a, b, k, min(r, k)))
    return out


def keep_heaviest(weights, budgets, groups=None, recent=0):
    """The rows that stay when each group is brought to its budget, int32, ascending.

    weights: float32 of P values (accumulated blend weights); groups: (begin, end) row
    ranges in ascending order, as merge_ply returns them (default: one group of all rows);
    budgets and recent: a whole number for all groups or a list with one for each.  A group of n
    rows keeps min(budget, n): its last `recent` ones and the heaviest of the others, of
    equals the lowest row; NaN counts as lighter than everything.  Rows in no group go."""
    _typed("keep_heaviest", weights=weights)
    P = weights.numel()
    if P >= 2 ** 31:
        raise RuntimeError("keep_heaviest: at most 2^31 - 1 weights")
    return _keep(weights, _keep_groups("keep_heaviest", P, budgets, groups, recent))


def _keep(weights, plan):
    """keep_heaviest of a finished plan (_keep_groups)."""
    P = weights.numel()
    _on_gpu("keep_heaviest", weights)
    weights = weights.contiguous()
    if _HOST is not None:
        return _HOST.keep_heaviest(weights, plan)
    _trace_check("keep_heaviest")
    ids = torch.empty(sum(k for _, _, k, _ in plan), dtype=torch.int32, device=weights.device)
    if ids.numel():
        ws = torch.empty(int(_lib.gsr_keep_ws_bytes(P)), dtype=torch.uint8, device=weights.device)
        _call(weights.device, _lib.gsr_keep_heaviest, P, weights.data_ptr(), len(plan), (_Group * len(plan))(*plan),
              ids.data_ptr(), ws.data_ptr())
    return ids


def take_rows(ids, tensors, out=None):
    """[t[ids] for t in tensors] in one launch: ids int32 [K], tensors contiguous float32 or
    int32 of any shape [rows, ...] on the same GPU; `out`, if given, contiguous tensors of
    K rows each that share no memory with the inputs.  An id outside a tensor gives a row of zeros.
    Not differentiable (like prune_points, it moves parameters and moments)."""
    _typed("take_rows", torch.int32, ids=ids)
    if ids.dim() != 1 or not ids.is_contiguous():
        raise RuntimeError("take_rows: ids must be contiguous, of shape (K,)")
    if ids.shape[0] >= 2 ** 31:
        raise RuntimeError("take_rows: at most 2^31 - 1 ids")
    return _take(ids, list(tensors), None if out is None else list(out), None)


def _take(ids, tensors, out, pad):
    K = ids.shape[0]
    if out is not None and len(out) != len(tensors):
        raise RuntimeError("take_rows: one output for each tensor")
    if _HOST is not None and ids.device.type == "cuda":
        try:
            got = _HOST.take_rows(ids, tensors, out or [], pad or [], out is not None)
            return got if out is None else out
        except TypeError:  # something that is no tensor: refused below
            pass
    _trace_check("take_rows")
    given = out is not None
    if out is None:
        out = [torch.empty((K,) + tuple(t.shape[1:]), dtype=t.dtype, device=t.device) if isinstance(t, torch.Tensor)
               else None for t in tensors]
    table = (_Rows * len(tensors))()
    for n, (t, o) in enumerate(zip(tensors, out)):
        for x, name in ((t, "tensors"), (o, "out")):
            if not isinstance(x, torch.Tensor) or x.dtype not in (torch.float32, torch.int32) or x.dim() < 1 or \
                    not x.is_contiguous() or x.device != ids.device or x.shape[0] >= 2 ** 31:
                raise RuntimeError(f"take_rows: {name}[{n}] must be a contiguous float32 or int32 tensor of rows on "
                                   f"{ids.device}")
        if o.dtype != t.dtype or o.shape[0] != K or o.shape[1:] != t.shape[1:]:
            raise RuntimeError(f"take_rows: out[{n}] must be {t.dtype} of {K} rows like tensors[{n}]")
        width = 1
        for d in t.shape[1:]:
            width *= d
        _width_check("take_rows", width)
        table[n] = (t.data_ptr(), o.data_ptr(), width, t.shape[0], pad[n] if pad else 0)
    _on_gpu("take_rows", ids)
    if tensors:
        _call(ids.device, _lib.gsr_take_rows, K, ids.data_ptr(), len(tensors), table)
    if given:
        for o in out:
            _written(o)
    return out


def take_gaussians(spec, ids, arenas):
    """The Gaussians `ids` (int32 [K]) of arenas laid out by `spec` (parameters, moments):
    (new ArenaSpec, [new arenas]), padding cleared."""
    new = _C.ArenaSpec(int(ids.shape[0]), spec.M, spec.C)
    outs = [torch.empty(new.total, dtype=torch.float32, device=ids.device) for _ in arenas]
    src, dst, pad = [], [], []
    for a, o in zip(arenas, outs):
        for b, name in enumerate(_C.BLOCK_NAMES):
            src.append(spec.block(a, name))
            dst.append(new.block(o, name))
            pad.append(new.off[b + 1] - new.off[b] - new.width[name] * new.P)
    _take(ids, src, dst, pad)
    return new, outs


# ---- a trained scene for rendering --------------------------------------------------------------
class CompactGaussians:
    """A GaussianModel as it is rendered after training, with the SH coefficients above the
    constant one in 4 bits: 90 bytes a Gaussian at degree 3 and two classes where the model's arena and
    activations take 284 (and its moments twice 244 more).  Made by GaussianModel.compact();
    offers what render() reads (get_xyz, get_colors, get_opacity, get_scaling,
    get_rotation, get_segment, get_features), all without gradients."""
    feature_bits = 4
    _TENSORS = ("xyz", "features_dc", "codes", "scales", "opacity", "scaling", "rotation", "segment")

    def __init__(self, xyz, features_dc, rest, opacity, scaling, rotation, segment, active_sh_degree):
        P = xyz.shape[0]
        if not isinstance(rest, MX4Rows) or rest.rows != P or rest.width % 3 or rest.width > 45:
            raise RuntimeError(f"CompactGaussians: rest must be MX4Rows of {P} rows of 3 (M - 1) values, M of 1..16")
        for t, name, cols in ((xyz, "xyz", 3), (opacity, "opacity", 1), (scaling, "scaling", 3),
                              (rotation, "rotation", 4)):
            if t.shape != (P, cols) or t.dtype != torch.float32:
                raise RuntimeError(f"CompactGaussians: {name} must be float32 of shape ({P}, {cols})")
        if features_dc.shape != (P, 1, 3) or segment.dim() != 2 or segment.shape[0] != P:
            raise RuntimeError(f"CompactGaussians: features_dc must be ({P}, 1, 3) and segment ({P}, classes)")
        if not 0 <= active_sh_degree <= 3 or (active_sh_degree + 1) ** 2 > rest.width // 3 + 1:
            raise RuntimeError("CompactGaussians: the features do not hold the active SH degree")
        self.get_xyz, self.features_dc, self.rest = xyz, features_dc, rest
        self.get_opacity, self.get_scaling, self.get_rotation, self.get_segment = opacity, scaling, rotation, segment
        self.active_sh_degree = int(active_sh_degree)
        self.max_sh_degree = {1: 0, 4: 1, 9: 2, 16: 3}.get(rest.width // 3 + 1, self.active_sh_degree)

    num_points = property(lambda self: self.get_xyz.shape[0])
    device = property(lambda self: self.get_xyz.device)
    num_class = property(lambda self: self.get_segment.shape[1])

    @property
    def nbytes(self):
        return sum(t.numel() * t.element_size() for t in self.state_dict().values() if isinstance(t, torch.Tensor))

    @property
    def get_features(self):
        """Decoded coefficients, float32 [P, M, 3]."""
        return torch.cat((self.features_dc, self.rest.dequantize().view(self.num_points, self.rest.width // 3, 3)), 1)

    @torch.no_grad()
    def get_colors(self, campos):
        """Colours seen from campos ([3] -> [P, 3], [V, 3] -> [V, P, 3])."""
        return sh_colors(self.get_xyz, self.features_dc, self.rest, campos, self.active_sh_degree)

    def state_dict(self):
        """Plain tensors and numbers (for torch.save; from_state_dict reads it)."""
        return {"xyz": self.get_xyz, "features_dc": self.features_dc, "codes": self.rest.codes,
                "scales": self.rest.scales, "opacity": self.get_opacity, "scaling": self.get_scaling,
                "rotation": self.get_rotation, "segment": self.get_segment, "rest_width": self.rest.width,
                "active_sh_degree": self.active_sh_degree}

    @classmethod
    def from_state_dict(cls, sd, device="cuda"):
        t = {k: sd[k].to(device).contiguous() for k in cls._TENSORS}
        return cls(t["xyz"], t["features_dc"], MX4Rows(t["codes"], t["scales"], sd["rest_width"]), t["opacity"],
                   t["scaling"], t["rotation"], t["segment"], int(sd["active_sh_degree"]))
