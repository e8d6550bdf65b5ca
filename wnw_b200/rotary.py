"""Rotary positions with one or several axes (``wnw_rotary``).

A decoder's rotation turns dimension i of a head with dimension i + rot / 2 by
position x inv_freq[i].  With several axes (time, height and width of image,
video and time-aligned audio tokens) every pair of dimensions follows one
axis' position.  Angles are computed in 64 bits from the integer positions, so
far positions keep their phase; the tensors are read and written once.

No reference counterpart: the reference leaves the rotation to the model
(src/common/adapters/voxtral.py:98-140).
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from wnw_b200 import native as N
from wnw_b200.kernels import LAUNCHES, check_device_error

_TYPES = (torch.float32, torch.float16, torch.bfloat16)


class Rotary:
    """One rotation: frequencies ``inv_freq`` [rot / 2] (fp32; taken as the
    exact numbers they are), the axis of each pair, and ``scaling`` on cosines
    and sines.  ``sections`` gives the pairs of each axis as consecutive runs
    ((16, 24, 24): 16 pairs for time, 24 for height, 24 for width); ``axes``
    names each pair's axis instead, for interleaved layouts.  Neither: one
    axis.  Dimensions beyond rot pass through.

    Calls may overlap on several streams; the handle holds constants and a
    device error word only (``check()`` reads it back), whose making must be
    ordered before its first use on another stream."""

    def __init__(self, inv_freq, sections=None, axes=None, scaling=1.0, device=None):
        inv_freq = torch.as_tensor(inv_freq, dtype=torch.float32, device=device).contiguous()
        if inv_freq.dim() != 1 or inv_freq.numel() == 0 or inv_freq.numel() % 8:
            raise ValueError(f"inv_freq {tuple(inv_freq.shape)}: a vector of a multiple of 8 frequencies")
        half = inv_freq.numel()
        if axes is not None and sections is not None:
            raise ValueError("give sections or axes, not both")
        if axes is None:
            sections = [half] if sections is None else [int(n) for n in sections]
            if any(n < 0 for n in sections) or sum(sections) != half:
                raise ValueError(f"sections {sections} do not add up to the {half} rotated pairs")
            axes = [a for a, n in enumerate(sections) for _ in range(n)]
            self.num_axes = len(sections)
        else:
            axes = [int(x) for x in axes]
            if len(axes) != half or min(axes) < 0:
                raise ValueError(f"axes must name an axis (>= 0) for each of the {half} rotated pairs")
            self.num_axes = max(axes) + 1
        if self.num_axes > 4:
            raise ValueError(f"{self.num_axes} axes: at most 4")
        self.rot_dim, self.scaling, self.device = 2 * half, float(scaling), inv_freq.device
        self.inv_freq = inv_freq
        self.axis = torch.tensor(axes, dtype=torch.int32, device=inv_freq.device)
        self.err = torch.zeros(1, dtype=torch.int32, device=inv_freq.device)
        self._index, self._calls = inv_freq.get_device(), {}  # argument blocks by geometry
        self._freq64 = inv_freq.double()
        self._freq_ptr, self._axis_ptr, self._err_ptr = (t.data_ptr() for t in (self._freq64, self.axis, self.err))

    def rope(self, positions, batch, tokens):
        """The ``wnw_rope`` for positions [axes, batch, tokens] (or [batch,
        tokens] for one axis), after checking them."""
        shape = positions.shape
        if len(shape) == 2 and self.num_axes == 1:
            positions = positions[None]
            shape = positions.shape
        if shape != (self.num_axes, batch, tokens):
            raise ValueError(f"positions {tuple(shape)}: expected {(self.num_axes, batch, tokens)}")
        t = positions.dtype
        if t is not torch.int64 and t is not torch.int32:
            raise TypeError(f"positions are int32 or int64, not {t}")
        return N.Rope(self.rot_dim, self.num_axes, self._freq_ptr, self._axis_ptr, positions.data_ptr(),
                      t is torch.int64, *positions.stride(), self.scaling)

    def __call__(self, q, k, positions, *, inverse=False, out=None, stream=None):
        """Rotated (q, k): q [B, Hq, n, D] and k [B, Hkv, n, D] (or None) of one
        type (fp32, fp16, bf16), rows contiguous and 16-byte aligned, other
        dimensions of any stride; positions [axes, B, n] ([B, n] with one
        axis), int32 or int64: below 2^29 in magnitude their angles are exact,
        above (up to 2^51) they carry a rounding to 64 bits.  ``inverse``
        applies the transposed rotation: the gradient of the forward one.
        ``out``: (q, k) to write, each of which may be its own input and shares
        no memory with the other tensors.  ``stream``: launch there, behind
        what the caller made it wait for.  Differentiable with respect to q and
        k, backward and forward (dual tensors)."""
        if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)) or _dual(q, k):
            if out is not None or stream is not None:
                raise ValueError("out and stream cannot be given where gradients are wanted")
            return _Rotate.apply(self, q, k, positions, inverse)
        if out is not None:
            plain(*out)
        return self._launch(q, k, positions, inverse, out, stream)

    def _launch(self, q, k, positions, inverse, out, stream):
        # checks and argument block depend on shapes, strides and types alone:
        # each geometry is looked at once, a call brings its pointers
        qo, ko = (None, None) if out is None else out
        key = (q.shape, q.stride(), q.dtype, positions.shape, positions.stride(), positions.dtype, bool(inverse),
               out is None, *(None if t is None else (t.shape, t.stride(), t.dtype) for t in (k, qo, ko)))
        base = self._calls.get(key)
        if base is None:
            base = self._call_args(q, k, positions, inverse, out)
            if len(self._calls) >= 64:
                self._calls.clear()
            self._calls[key] = base
        index = self._index
        if out is not None:
            base[2](qo.data_ptr(), q.data_ptr(), None if ko is None else ko.data_ptr(),
                    None if k is None else k.data_ptr())
        if out is None:
            qo = made_on(stream, index, torch.empty_like, q, memory_format=torch.contiguous_format)
            if k is not None:
                ko = made_on(stream, index, torch.empty_like, k, memory_format=torch.contiguous_format)
        for t in (q, k, positions, qo, ko):
            if t is not None and (t.get_device() != index or index < 0):
                raise ValueError(f"a tensor on {t.device}: the rotation is on {self.device} and needs a CUDA device")
        launch(index, stream, _ROTARY, "wnw_rotary_step", base[1], q.data_ptr(), qo.data_ptr(),
               None if k is None else k.data_ptr(), None if ko is None else ko.data_ptr(), positions.data_ptr())
        if out is not None:
            written((qo,) if ko is None else (qo, ko))
        if stream is not None:
            keep_for(stream, q, k, qo, ko, positions, self._freq64, self.axis, self.err)
        return qo, ko

    def _call_args(self, q, k, positions, inverse, out):
        """(argument block without pointers, a reference to it, the check of
        given outputs' addresses) of one geometry, checked."""
        if q.dim() != 4 or q.dtype not in _TYPES:
            raise ValueError(f"q {tuple(q.shape)} {q.dtype}: expected [B, heads, n, D] in fp32, fp16 or bf16")
        B, Hq, n, D = q.shape
        if k is not None and (k.dim() != 4 or k.shape[0] != B or k.shape[2] != n or k.shape[3] != D
                              or k.dtype != q.dtype):
            raise ValueError(f"k {tuple(k.shape)} {k.dtype} does not go with q {tuple(q.shape)} {q.dtype}")
        if self.rot_dim > D:
            raise ValueError(f"{self.rot_dim} rotated dimensions in heads of {D}")
        strides = []
        for i, x in enumerate((q, k)):
            if x is None:
                if out is not None and out[i] is not None:
                    raise ValueError("out must match q and k in shape, type and device")
                strides += _NO_ROWS * 2
                continue
            if out is None:
                to = (None, *dense(x.shape))
            elif out[i] is None or out[i].shape != x.shape or out[i].dtype != x.dtype:
                raise ValueError("out must match q and k in shape, type and device")
            else:
                to = rows(out[i], "out", x.shape)
                distinct(out[i], "out")
            strides += (*rows(x, "qk"[i], x.shape), *to)
        a = N.RotaryArgs(N.dtype_code(q.dtype), D, B, n, Hq, 0 if k is None else k.shape[1], *strides,
                         self.rope(positions, B, n), bool(inverse), self._err_ptr)
        return a, C.byref(a), None if out is None else Apart(("q_out", out[0], q), ("k_out", out[1], k))

    def check(self):
        check_device_error(self.err)


class _Rotate(torch.autograd.Function):
    """The rotation is linear: its gradient is the transposed rotation, its
    forward derivative the rotation of the tangents."""

    @staticmethod
    def forward(ctx, rotary, q, k, positions, inverse):
        ctx.rotary, ctx.inverse = rotary, inverse
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)
        ctx.positions = positions
        out = rotary._launch(q, k, positions, inverse, None, None)
        ctx.like = [None if y is None else (y.shape, y.dtype, y.device) for y in out]
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        pos, = ctx.saved_tensors
        gq, gk = (g if need else None for g, need in zip((gq, gk), ctx.needs_input_grad[1:3]))
        return None, *_some(ctx.rotary, gq, gk, pos, not ctx.inverse), None, None

    @staticmethod
    def jvp(ctx, _rotary, tq, tk, _positions, _inverse):
        turned = _some(ctx.rotary, tq, tk, ctx.positions, ctx.inverse)
        # (an output whose input has no tangent is given a zero one: autograd takes no None for it)
        return tuple(t if t is not None or y is None else torch.zeros(y[0], dtype=y[1], device=y[2])
                     for t, y in zip(turned, ctx.like))


def _dual(*tensors):
    """Whether one of them carries a forward derivative."""
    return forward_ad._current_level >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _some(rotary, q, k, positions, inverse):
    """The rotation of derivatives, either of which may be None."""
    if q is not None:
        return rotary._launch(_rows(q), None if k is None else _rows(k), positions, inverse, None, None)
    if k is not None:
        return None, rotary._launch(_rows(k), None, positions, inverse, None, None)[0]
    return None, None


def _rows(x):
    """A gradient with rows that the kernel takes (broadcast ones are laid out)."""
    e = 4 if x.dtype == torch.float32 else 8
    if x.stride(3) != 1 or any(s % e for s in x.stride()[:3]) or x.data_ptr() % 16:
        return x.contiguous()
    return x


_NO_ROWS = (None, 0, 0, 0)


def rows(t, name, shape):
    """(pointer, batch, head and token strides) of [B, heads, n, D] rows."""
    sb, sh, sn, sd = t.stride()
    B, H, n, D = shape
    if sd != 1 and D > 1:
        raise ValueError(f"{name}: the head dimension must be contiguous (strides {t.stride()})")
    # a dimension of one may carry any stride
    return t.data_ptr(), sb if B > 1 else 0, sh if H > 1 else 0, sn if n > 1 else 0


def distinct(t, name):
    """Refuse an output whose elements share memory (an expanded one, say)."""
    span = 1
    for stride, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if stride < span:
            raise ValueError(f"{name}: elements share memory (shape {tuple(t.shape)}, strides {t.stride()})")
        span = stride * n


class Apart:
    """Refuses the outputs of one geometry's calls that share memory with
    another output, with another's input, or with their own at other elements.
    From (name, output, its input) tensors; a call brings their addresses, in
    the same order, None where there is no tensor."""

    def __init__(self, *triples):
        layouts = [(name, w, t) for name, *ts in triples for w, t in zip((True, False), ts)]
        self._pairs = []
        for j, (_, wj, b) in enumerate(layouts):
            for i, (name, wi, a) in enumerate(layouts[:j]):
                if a is None or b is None or not (wi or wj) or not (a.numel() and b.numel()):
                    continue
                own = i == j - 1 and j % 2 == 1 and all(
                    s == t or n == 1 for s, t, n in zip(a.stride(), b.stride(), a.shape))
                la, lb = ((tuple(t.shape), t.stride(), t.element_size()) for t in (a, b))
                self._pairs.append((i, j, _span(la), _span(lb), own, la, lb, name))

    def __call__(self, *at):
        seen = []  # (in place, several pairs are the same two)
        for i, j, after, before, own, la, lb, name in self._pairs:
            d = at[j] - at[i]
            if -before < d < after and not (own and d == 0) and (la, lb, d) not in seen:
                if _meet(la, lb, d):
                    raise ValueError(f"{name}: shares memory with another tensor of the call")
                seen.append((la, lb, d))


def _span(layout):
    shape, strides, size = layout
    return size * (1 + sum(s * (n - 1) for s, n in zip(strides, shape)))


def _meet(a, b, distance):
    """Whether two tensors (shape, strides, bytes an element) whose starts are
    so many bytes apart have an element in common, given that what they span
    does.  Exact where the strides are the same (views of one buffer), else
    taken to be so."""
    (na, sa, e), (nb, sb, f) = a, b
    if e != f or distance % e or len(na) != len(nb) \
            or any(x > 1 and y > 1 and s != t for s, t, x, y in zip(sa, sb, na, nb)):
        return True
    # a's element i and b's element j are one where the sum of stride x (i - j) is the distance of their starts
    dims = sorted(((s if x > 1 else t, y - 1, x - 1) for s, t, x, y in zip(sa, sb, na, nb) if x > 1 or y > 1),
                  reverse=True)

    def reach(at, rest):
        if at == len(dims) or dims[at][0] == 0:
            return rest == 0
        stride, down, up = dims[at]
        low, high = (sum(d[0] * d[w] for d in dims[at + 1:]) for w in (1, 2))
        first, last = -((high - rest) // stride), (rest + low) // stride
        return any(reach(at + 1, rest - stride * i) for i in range(max(first, -down), min(last, up) + 1))

    return reach(0, distance // e)


def dense(shape):
    """(batch, head, token) strides of a contiguous [B, heads, n, D]."""
    B, H, n, D = shape
    return H * n * D, n * D, D


_ROTARY = N.lib.wnw_rotary_step
_get_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def launch(index, stream, fn, name, *args):
    """Call an entry point with device ``index`` current, on ``stream`` or its
    current stream; a non-OK status raises."""
    if stream is not None and stream.device_index != index:
        raise ValueError(f"a stream of {stream.device}: the tensors are on CUDA device {index}")
    if _get_device() != index:
        with torch.cuda.device(index):
            return launch(index, stream, fn, name, *args)
    st = fn(*args, _raw_stream(index) if stream is None else stream.cuda_stream)
    if st:
        N.check(st, name)
    LAUNCHES[0] += 1


def made_on(stream, index, make, *args, **kw):
    """A result for a launch on ``stream`` (None: the current one): memory of
    that stream's, so that no earlier user of it on another stream is still at
    it, kept for the current stream too."""
    if stream is None:
        return make(*args, **kw)
    with torch.cuda.stream(stream):
        t = make(*args, **kw)
    if t.is_cuda:
        t.record_stream(torch.cuda.current_stream(index))
    return t


def plain(a, b=None):
    """Refuse to write into tensors that carry derivatives: the call would not
    be part of them."""
    wanted = a is not None and a.requires_grad or b is not None and b.requires_grad
    if wanted and torch.is_grad_enabled() or forward_ad._current_level >= 0 and _dual(a, b):
        raise ValueError("a given output carries derivatives: write into a detached one, or under no_grad")


#: tells autograd that a launch has written into the caller's tensors: what was
#: saved of them for a backward pass is refused there
written = increment_version


def keep_for(stream, *tensors):
    """Tensors of the current stream stay alive for launches on another one."""
    for t in tensors:
        if t is not None:
            t.record_stream(stream)
