"""The gated delta rule on the MI355X (``gpx_delta_*``): regression over a stream.

No counterpart in the reference, and no estimator of this package calls it: it is for programs that keep such a state of
their own.  By its method it is the exact GP's streaming relative: the GP solves for all targets at once in O(n^3), this
keeps one dk x dv map from keys to values and corrects it by the error of every token, in order, while it forgets --
for each sequence and head

    Sbar = exp(g) S;   e = v - Sbar^T k;   S <- Sbar + beta k e^T;   o = scale S^T q

Shapes: q, k (B, T, Hk, dk); v, o (B, T, Hv, dv), Hv a multiple of Hk (value head i reads key head
i // (Hv // Hk)); g (the LOG of the decay, at most 0, -inf forgets everything; growth, g > 0, costs as many bits as it
multiplies in 64 tokens) and beta (B, T, Hv) in float32; states (sequences, Hv, dk, dv) in float32.  q, k, v, o: float32, float16 or bfloat16, one type, sums in float32.
1 <= dk <= 128, 1 <= dv <= 1024, any T.  Any strides; q, k, v with a last dimension that is not dense are copied first.

Gradients are functions of their own, as everywhere in this package: nothing is recorded behind the
caller's back, so a forward and a backward call may be captured into a graph together.  Tensors that require a gradient are
therefore refused where torch records (RuntimeError); pass them detached, or call under torch.no_grad()."""
import ctypes as C

from . import _lib
from .device import ptr, tensor_runtime
from .orthogonal import check_tensor, type_id


SIZE_MAX = 1 << 30   # the library's sizes are 32-bit


def _dense(t):
    """t, or a packed copy where its last dimension is not dense or its tokens lie too far apart for the library."""
    return t if (t.stride(-1) == 1 or t.shape[-1] == 1) and t.stride(-3) <= 1 << 22 else t.contiguous()


def _dense_row(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _st(t):
    """{batch, token, head} strides; a dimension of one has none."""
    a, b, c = t.shape[:3]
    x, y, z = t.stride()[:3]
    return (x if a > 1 else 0, y if b > 1 else 0, z if c > 1 else 0)


def _st_row(t):
    """The same of a (batch, head) tensor of one token each."""
    a, c = t.shape[:2]
    x, z = t.stride()[:2]
    return (x if a > 1 else 0, 0, z if c > 1 else 0)


def _opt(t):
    return ptr(t) if t is not None else None


def _check(q, k, v, g, beta, dims):
    """(type number, key heads, dk, value heads, dv) of inputs that fit together."""
    import torch
    Tensor = torch.Tensor
    if not (isinstance(q, Tensor) and isinstance(k, Tensor) and isinstance(v, Tensor) and isinstance(g, Tensor)
            and isinstance(beta, Tensor)):
        for name, t in (("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta)):
            check_tensor(t, name)
    kind = q.dtype
    dtype = type_id(q)
    if not dtype:   # float64 has number 0
        raise TypeError("element type %s is not one of float32, float16, bfloat16" % kind)
    if k.dtype != kind or v.dtype != kind:
        raise TypeError("q, k and v must have one type")
    if g.dtype != torch.float32 or beta.dtype != torch.float32:
        raise TypeError("g and beta must be float32")
    qs, vs = q.shape, v.shape
    if len(qs) != dims or len(vs) != dims:
        raise ValueError("q, k and v must have %d dimensions" % dims)
    if k.shape != qs:
        raise ValueError("q and k must have the same shape")
    if vs[:-2] != qs[:-2] or g.shape != vs[:-1] or beta.shape != vs[:-1]:
        raise ValueError("q, k, v, g and beta do not agree in batch, tokens or value heads")
    Hk, dk = qs[-2:]
    Hv, dv = vs[-2:]
    if Hk < 1 or Hv < 1 or Hv % Hk:
        raise ValueError("the value heads (%d) must be a multiple of the key heads (%d)" % (Hv, Hk))
    if max(qs) > SIZE_MAX or max(vs) > SIZE_MAX:
        raise ValueError("a size of q, k or v is beyond 2^30")
    if not 1 <= dk <= 128 or not 1 <= dv <= 1024:
        raise ValueError("dk = %d must be in [1, 128], dv = %d in [1, 1024]" % (dk, dv))
    return dtype, Hk, dk, Hv, dv


def _check_state(t, shape, name):
    import torch
    if t is None:
        return
    check_tensor(t, name)
    if t.dtype != torch.float32 or t.shape != shape:
        raise ValueError("%s must be float32 of shape %s" % (name, tuple(shape)))
    if not t.data_ptr() and t.numel():   # the library takes no address for no state
        raise ValueError("%s has no memory" % name)


def _aligned(t):
    """t, or a packed copy where the library's 16-byte accesses to states would not fit."""
    import torch
    if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _bytes(rt, d, use):
    """A workspace of the library, and its size."""
    size = int(rt.lib.gpx_delta_work_bytes(C.byref(d), use))
    return rt.torch.empty(max(size, 256), dtype=rt.torch.uint8, device=rt.dev), size


def _version(t):
    return None if t.is_inference() else t._version   # inference tensors do not count their writes


def _place(t):
    """What changes when t is written, moved or given up."""
    return _version(t), t.data_ptr(), t.untyped_storage().nbytes()


class Saved:
    """What a forward call keeps for its backward call."""

    def __init__(self, desc, inputs, state, work, stream):
        self.desc, self.has_state, self.work, self.stream = desc, state is not None, work, stream
        # aliases, which hold the memory that desc points to: a caller's tensor may be given other memory (t.data = ...)
        self.inputs = [t.detach() for t in inputs]
        self.places = [_place(t) for t in self.inputs]

    def check(self):
        if [_place(t) for t in self.inputs] != self.places:
            raise RuntimeError("an input of the forward call has been modified in place, or its memory resized, since")


def gated_delta_rule(q, k, v, g, beta, initial_state=None, cu_seqlens=None, scale=None, save_for_backward=False):
    """(o, final_state), and with ``save_for_backward`` also what ``gated_delta_rule_backward`` needs.

    cu_seqlens: None, each batch row is a sequence; or B = 1 and an int32 tensor on the device of n + 1 ends of packed
    sequences (sequence s is tokens cu_seqlens[s] to cu_seqlens[s + 1]; empty ones pass their state through).  Values
    outside [0, T] are clamped and a decreasing one is read as the one before it; outputs of tokens that belong
    to no sequence are zeros.  initial_state: (sequences, Hv, dk, dv) float32, None for zeros.  scale: dk ** -0.5 by default.

    Long inputs run in chunks of 64 tokens on the matrix cores, up to 16 tokens go through the recurrence.  There a NaN or an
    infinity in a token's inputs may reach the tokens before it in its chunk, besides the later ones of its sequence and head that
    it reaches in any case; never earlier chunks, other sequences or heads.  Asynchronous
    on the current stream; may be captured into a graph after one call outside."""
    import torch
    dtype, Hk, dk, Hv, dv = _check(q, k, v, g, beta, 4)
    B, T = q.shape[:2]
    sequences = 0
    if cu_seqlens is not None:
        check_tensor(cu_seqlens, "cu_seqlens")
        if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2:
            raise ValueError("cu_seqlens must be a one-dimensional int32 tensor of at least two values")
        if B != 1:
            raise ValueError("packed sequences need a batch of one")
        sequences = cu_seqlens.numel() - 1
        if sequences > SIZE_MAX:
            raise ValueError("%d sequences are too many" % sequences)
    shape = (sequences or B, Hv, dk, dv)
    _check_state(initial_state, shape, "initial_state")
    rt = tensor_runtime(q, k, v, g, beta, initial_state, cu_seqlens)
    with rt.current_stream():
        q, k, v = _dense(q), _dense(k), _dense(v)
        if cu_seqlens is not None:
            cu_seqlens = cu_seqlens.contiguous()
        state = _aligned(initial_state)
        d = _lib.Delta(dtype, B, T, sequences, Hk, Hv, dk, dv, dk ** -0.5 if scale is None else float(scale),
                       cu_seqlens.data_ptr() if sequences else None, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(),
                       beta.data_ptr(), _st(q), _st(k), _st(v), _st(g), _st(beta))
        o = (torch.zeros if sequences else torch.empty)((B, T, Hv, dv), dtype=q.dtype, device=q.device)
        final = torch.empty(shape, dtype=torch.float32, device=q.device)
        work, size = _bytes(rt, d, 3 if save_for_backward else 0)
        saved, kept = _bytes(rt, d, 1) if save_for_backward else (None, 0)
        _lib.check(rt.lib.gpx_delta_forward(rt.h, C.byref(d), _opt(state), ptr(o), ptr(final), ptr(work), size, _opt(saved), kept),
                   "gpx_delta_forward")
    if not save_for_backward:
        return o, final
    inputs = [t for t in (q, k, v, g, beta, cu_seqlens) if t is not None]
    return o, final, Saved(d, inputs, initial_state, saved, torch.cuda.current_stream(q.device))


def gated_delta_rule_backward(saved, d_o, d_final_state=None):
    """(d_q, d_k, d_v, d_g, d_beta, d_initial_state) of sum(d_o * o) + sum(d_final_state * final_state).

    ``saved`` comes from the forward call; it is only read, so the call may be repeated with other d_o.  It holds the memory of the
    forward call's inputs; RuntimeError if they have been written or their storage resized in between.  d_q, d_k, d_v have the type of
    q, k, v, the others float32; d_initial_state is None if the forward call had no initial_state.  Tokens that belong
    to no sequence get zeros."""
    import torch
    if not isinstance(saved, Saved):
        raise TypeError("saved must come from gated_delta_rule(..., save_for_backward=True)")
    saved.check()
    q, k, v, g, beta = saved.inputs[:5]
    d = saved.desc
    check_tensor(d_o, "d_o")
    if d_o.shape != v.shape or d_o.dtype != v.dtype:
        raise ValueError("d_o must have the shape and the type of o")
    shape = (d.sequences or d.batch, d.value_heads, d.dk, d.dv)
    _check_state(d_final_state, shape, "d_final_state")
    rt = tensor_runtime(q, d_o, d_final_state)
    stream = torch.cuda.current_stream(q.device)
    if stream != saved.stream:   # what the forward call allocated may be dropped while this stream still reads it
        for t in (*saved.inputs, saved.work):
            t.record_stream(stream)
    with rt.current_stream():
        d_o, d_final = _dense(d_o), _aligned(d_final_state)
        new = torch.zeros if d.sequences else torch.empty
        grads = [new(t.shape, dtype=t.dtype, device=q.device) for t in (q, k, v, g, beta)]
        d_state = torch.empty(shape, dtype=torch.float32, device=q.device) if saved.has_state else None
        scratch, size = _bytes(rt, d, 2)
        st = _lib.Strided(*_st(d_o))
        _lib.check(rt.lib.gpx_delta_backward(rt.h, C.byref(d), ptr(d_o), C.byref(st), _opt(d_final), *map(ptr, grads), _opt(d_state),
                                             ptr(saved.work), saved.work.numel(), ptr(scratch), size), "gpx_delta_backward")
    return (*grads, d_state)


# What a step of these types, shapes and strides has been found to be.  A decoder makes the same call for every token, and the
# checks and the description take as long as the rest of the call (13.5 us with them).
_known_steps = {}


def _step_description(q, k, v, g, beta, state, slots, state_out, scale):
    """(the bytes of a gpx_delta without its pointers, whether q, k, v are used as they are, o's shape) of a valid step."""
    import torch
    dtype, Hk, dk, Hv, dv = _check(q, k, v, g, beta, 3)
    B = q.shape[0]
    check_tensor(state, "state")
    n = state.shape[0] if state.dim() else 0
    if n > SIZE_MAX:
        raise ValueError("%d states are too many" % n)
    _check_state(state, (n, Hv, dk, dv), "state")
    if slots is None:
        if n != B:
            raise ValueError("%d states for %d rows: name them with slots" % (n, B))
    else:
        check_tensor(slots, "slots")
        if slots.dtype != torch.int32 or tuple(slots.shape) != (B,):
            raise ValueError("slots must be an int32 tensor with one value per row")
    _check_state(state_out, state.shape, "state_out")
    if not state.is_contiguous() or not state_out.is_contiguous():
        raise ValueError("state and state_out must be packed")
    as_used = [_dense_row(t) for t in (q, k, v)]
    dense = all(a is b for a, b in zip(as_used, (q, k, v)))
    d = _lib.Delta(dtype, B, 1, 0, Hk, Hv, dk, dv, dk ** -0.5 if scale is None else scale, None, None, None, None, None, None,
                   *map(_st_row, as_used), _st_row(g), _st_row(beta))
    return bytes(d), dense, (B, Hv, dv)


def gated_delta_rule_step(q, k, v, g, beta, state, slots=None, state_out=None, scale=None):
    """One token for each of B rows: q, k (B, Hk, dk); v (B, Hv, dv); g, beta (B, Hv).  Returns (o, state_out).

    state: (n, Hv, dk, dv) float32, packed, n = B unless ``slots`` names the state of each row (int32 tensor on the device).
    It is updated in place unless ``state_out`` (its shape, no other view of its memory) is given.  A row whose slot
    is outside [0, n) is padding: its o is zero and no state is written for it; states that no row names are not touched.  Rows with
    the same slot are taken in their order, as successive tokens of one sequence."""
    import torch
    if state_out is None:
        state_out = state
    if scale is not None:
        scale = float(scale)
    try:
        key = (scale, q.dtype, q.shape, q.stride(), k.dtype, k.shape, k.stride(), v.dtype, v.shape, v.stride(), g.dtype, g.shape,
               g.stride(), beta.dtype, beta.shape, beta.stride(), state.dtype, state.shape, state.stride(), state_out.dtype,
               state_out.shape, state_out.stride(), slots if slots is None else (slots.dtype, slots.shape))
        known = _known_steps.get(key)
    except (AttributeError, TypeError):   # not tensors: _step_description says which
        key = known = None
    if known is None:
        known = _step_description(q, k, v, g, beta, state, slots, state_out, scale)
        if len(_known_steps) >= 256:
            _known_steps.clear()
        if key is not None:
            _known_steps[key] = known
    at, to = state.data_ptr(), state_out.data_ptr()
    if not (at and to) and state.numel():
        raise ValueError("state or state_out has no memory")
    if 0 < abs(to - at) < state.numel() * 4:
        raise ValueError("state_out overlaps state")
    rt = tensor_runtime(q, k, v, g, beta, state, slots, state_out)
    with rt.current_stream():
        description, dense, shape = known
        if not dense:
            q, k, v = _dense_row(q), _dense_row(k), _dense_row(v)
        if slots is not None:
            slots = slots.contiguous()
        o = (torch.empty if slots is None else torch.zeros)(shape, dtype=q.dtype, device=q.device)
        d = _lib.Delta.from_buffer_copy(description)
        d.q, d.k, d.v, d.g, d.beta = q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr()
        rc = rt.lib.gpx_delta_step(rt.h, C.byref(d), state.shape[0], _opt(slots), at, to, o.data_ptr())
        if rc:
            _lib.check(rc, "gpx_delta_step")
        torch.autograd.graph.increment_version(state_out)   # written behind torch's back: what was saved of it is stale
    return o, state_out
