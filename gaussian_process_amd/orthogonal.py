"""Orthogonalisation of matrix-shaped updates on the MI355X (``gpx_orthogonalize``).

No counterpart in the reference, whose parameters are scalars and length scales that L-BFGS-B moves (base.py:21-58), as
are those of the estimators here: none of them calls it.  It is for programs that train matrices of their own."""
import ctypes as C
import math

from . import _lib
from .device import ptr, tensor_runtime

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


_ids = {}


def type_id(t):
    """gpx's number of a tensor's element type; None if it has none."""
    try:
        return _ids[t.dtype]
    except KeyError:
        return _ids.setdefault(t.dtype, _lib.GPX_TYPE.get(str(t.dtype).replace("torch.", "")))


def check_tensor(t, name):
    import torch
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch tensor, got %s" % (name, type(t).__name__))
    return t


def _stack(t):
    """(..., n, m) -> a (batch, n, m) view, or None where the leading dimensions have no common stride."""
    try:
        return t.view(math.prod(t.shape[:-2]), *t.shape[-2:])
    except RuntimeError:
        return None


def _strides(t):
    return _lib.Strided(*(t.stride(d) if t.shape[d] > 1 else 0 for d in range(2)), t.stride(2))


def _overlap(t):
    """Whether two elements of t share memory (an expanded dimension): such a tensor cannot be written."""
    dims = sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz > 1)
    reach = 0
    for st, sz in dims:
        if st <= reach:
            return True
        reach += st * (sz - 1)
    return False


def orthogonalize(G, steps=5, coefficients=COEFFICIENTS, eps=1e-7, alpha=1.0, beta=0.0, base=None, out=None, reduced=False):
    """out = alpha * O + beta * base with O the (nearly) orthogonal factor of G by Newton-Schulz products:

        X = G / (|G|_F + eps);  steps times:  A = X X^T,  B = b A + c A A,  X = a X + B X;  O = X

    (a, b, c) = ``coefficients``.  The default ones push every singular value of a generic G into about [0.7, 1.2]
    within five steps; (1.5, -0.5, 0) converges to the polar factor itself, more slowly.

    G: (..., n, m) tensor on the MI355X, float64, float32, float16 or bfloat16, any strides (a transposed view costs
    nothing); leading dimensions are a stack of matrices, each with a norm of its own.  ``base`` (needed when beta != 0) and ``out``
    have G's shape and type; ``out`` may be ``base`` or ``G`` itself: ``orthogonalize(G, alpha=-lr, beta=1 - lr * decay,
    base=W, out=W)`` is an optimiser's update.  Returns out.  No gradient is recorded: tensors that require one are refused
    (RuntimeError) outside torch.no_grad(), as torch does with writes to a leaf.

    float64 is computed in float64; the other types on the fp16 matrix cores with float32 sums and 22 bits per intermediate
    value.  ``reduced`` (bfloat16 only) makes do with 11 bits, which takes a third of the products; the result's error is then 1.03 to
    1.23 times that of rounding the exact result (1024 x 1024 to 130 x 260), and 1.00 times without.  A matrix of zeros gives zeros
    (NaNs with eps = 0), one with a NaN or an infinity NaNs.  Of values below 2^-28 of the spectrum's bound, such as all of a matrix whose
    norm is below 1e-4 eps, bits are lost outside float64; in float64 the squares of G must be normal numbers.  Asynchronous on
    the current stream; may be captured into a graph after one call outside."""
    import torch
    check_tensor(G, "G")
    dtype = type_id(G)
    if dtype is None:
        raise TypeError("element type %s is not one of %s" % (G.dtype, ", ".join(_lib.GPX_TYPE)))
    if G.dim() < 2:
        raise ValueError("G must have at least two dimensions")
    if max(math.prod(G.shape[:-2]), *G.shape[-2:]) > 65536:   # before the library's 32-bit sizes cut it off
        raise ValueError("G has more than 65535 matrices or 65536 rows or columns")
    if reduced and G.dtype != torch.bfloat16:
        raise ValueError("reduced is for bfloat16")
    if beta != 0.0 and base is None:
        raise ValueError("beta != 0 needs base")
    for name, t in (("base", base), ("out", out)):
        if t is None:
            continue
        check_tensor(t, name)
        if t.shape != G.shape or t.dtype != G.dtype:
            raise ValueError("%s must have the shape and the type of G" % name)
    if len(coefficients) != 3:
        raise ValueError("coefficients are three numbers (a, b, c)")
    if out is not None and _overlap(out):
        raise ValueError("elements of out share memory")
    if beta == 0.0:
        base = None
    rt = tensor_runtime(G, base, out)
    if out is None:
        out = torch.empty_like(G, memory_format=torch.contiguous_format)
    o3 = _stack(out)
    if o3 is None:
        raise ValueError("the leading dimensions of out have no common stride")
    g3 = _stack(G)
    if g3 is None:
        g3 = _stack(G.contiguous())
    b3 = None
    if base is not None:
        same = base.data_ptr() == out.data_ptr() and base.stride() == out.stride()
        if not same and base.untyped_storage().data_ptr() == out.untyped_storage().data_ptr():
            base = base.clone()   # another view of out's memory: read it before out is written
        b3 = _stack(base)
        if b3 is None:
            b3 = _stack(base.contiguous())
    batch, n, m = g3.shape
    if G.dtype == torch.bfloat16 and not reduced:
        dtype |= _lib.GPX_TWO_PLANES
    with rt.current_stream():
        size = int(rt.lib.gpx_orthogonalize_work_bytes(dtype, batch, n, m))
        work = torch.empty(max(size, 16), dtype=torch.uint8, device=G.device)
        _, coef = _keep = _lib.host_doubles(coefficients)
        gs, os_ = _strides(g3), _strides(o3)
        bs = _strides(b3) if b3 is not None else None
        _lib.check(rt.lib.gpx_orthogonalize(
            rt.h, dtype, batch, n, m, ptr(g3), C.byref(gs), int(steps), coef, float(eps), float(alpha), float(beta),
            ptr(b3) if b3 is not None else None, C.byref(bs) if bs is not None else None, ptr(o3), C.byref(os_),
            ptr(work), size), "gpx_orthogonalize")
        torch.autograd.graph.increment_version(out)   # written behind torch's back: what was saved of it is stale
    return out
