"""A paged key/value cache and the two operators of a serving step around it.

* :func:`rotate_append` turns new queries and keys by their positions (rotary
  positions of one or several axes) and writes keys and values to the cache;
* :func:`attention` is the attention of a ragged chunk of new tokens, one token
  a sequence (decoding) upwards, over that cache.

A cache is two tensors, keys and values, of shape [pages, page_size, kv_heads,
head_dim] with any strides of the outer dimensions, so ``[pages, kv_heads,
page_size, head_dim]`` storage is passed as its ``transpose(1, 2)``.  Both
operators run on the current stream of their tensors' device, or on the CUDA
stream ``stream`` (its address; it has to last as long as what was allocated for
calls on it: returned tensors, plans, rotations), and return without waiting.
Tensors that they return may be used on that stream and on the current one;
those that they are given are the caller's to keep until a ``stream`` is through
with them.  They are thin over the C ABI (``emmy_rotate_append``,
``emmy_paged_attention`` in ``include/emmy_b200.h``) and raise
:class:`~.native.EmmyError` with its message on arguments it refuses,
``ValueError`` on what only Python can see.  They have no backward pass, and
refuse tensors that require grad unless gradients are off.
"""
from __future__ import annotations

import ctypes
import struct

import torch

from . import native

_DTYPES = {torch.float16: 6, torch.float32: 7, torch.bfloat16: 9}

# the argument structures of the C ABI, packed in one go: 1 us against 6 for a
# ctypes structure of as many fields, on calls of 3 us on the GPU
_ROTATE_APPEND_ARGS = struct.Struct("@10i10Q15q")
_ATTENTION_ARGS = struct.Struct("@4if8Q11q")

_i32 = ctypes.c_int32
_CONTIGUOUS = torch.contiguous_format


class _PlanArgs(ctypes.Structure):
    _fields_ = [("sequences", _i32), ("q_lens", ctypes.c_void_p), ("kv_lens", ctypes.c_void_p),
                ("q_heads", _i32), ("kv_heads", _i32), ("head_dim", _i32), ("causal", _i32), ("window", _i32),
                ("ctas", _i32)]


def _need(ok, text):
    if not ok:
        raise ValueError(text)


def _check(name, t, ndim, dtype, device):
    """A tensor of the cache operators: on the GPU, its innermost stride 1.  The
    operators look all of theirs over in one expression first (a call of 3 us on the
    GPU would wait for the host otherwise) and come here for the reason."""
    if not isinstance(t, torch.Tensor) or t.ndim != ndim:
        raise ValueError(f"{name}: a tensor of {ndim} dimensions is wanted")
    if t.dtype is not dtype:
        raise ValueError(f"{name}: {dtype} is wanted, not {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name}: on {t.device}, not on {device}")
    stride = t.stride()
    if stride[-1] != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}: the innermost stride must be 1")
    return stride


def _no_backward():
    """For serving: the results would be cut off from what made them without a word."""
    raise ValueError("a tensor requires grad, and this operator has no backward pass: call it under torch.no_grad()")


# what every call asks (of a device that is up: its tensors are there)
_grads_on, _empty_like = torch.is_grad_enabled, torch.empty_like
_current_device, _current_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
# as any operation in place does: autograd checks what it keeps by it
_written_to = torch.autograd.graph.increment_version


def _unfit(e):
    return ValueError(f"an argument does not fit its field of the C ABI: {e}")


def _cuda_device(name, t):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name}: a CUDA tensor is wanted")
    return t.device


_fns = {}


def _call(name, index, stream, *args):
    """One C-ABI call on ``stream`` with its device ``index`` current."""
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = getattr(native.lib(), name)
    if index != _current_device():
        with torch.cuda.device(index):
            return _call(name, index, stream, *args)
    rc = fn(*args, stream)
    if rc:
        native.check(rc)


def _stream_at(handle, device):
    # 0 and 1 are the default stream; ExternalStream(0) is one of PyTorch's pool
    return torch.cuda.default_stream(device) if handle in (0, 1) else torch.cuda.ExternalStream(handle, device=device)


def _made_for(stream, t):
    """Memory allocated here and used on another stream is not reused before that stream is through."""
    t.record_stream(_stream_at(stream, t.device))


def _new(stream, like, shape, dtype):
    """Memory for a result that the stream writes: its own, for what the current stream
    had there before may still run; the caller's, on the current stream, as well."""
    current = torch.cuda.current_stream(like.device)
    with torch.cuda.stream(_stream_at(stream, like.device)):
        t = like.new_empty(shape, dtype=dtype)
    t.record_stream(current)
    return t


class _Kept:
    """Device memory that calls on any stream use and that may be dropped while they run."""

    def _keep(self, *tensors, own=False):
        # own: allocated on the current stream just now; others may come from any
        self._tensors = [t for t in tensors if t is not None]
        self._streams = set()
        current = torch._C._cuda_getCurrentRawStream(tensors[0].device.index)
        if own:
            self._streams.add(current)
        else:
            self._used_on(current)

    def _used_on(self, stream):
        for t in self._tensors:
            _made_for(stream, t)
        self._streams.add(stream)


class Rotation(_Kept):
    """Rotary positions: ``frequencies`` (float32, on the GPU) has the radians
    per position of each pair, so its length is half of the components that
    turn, the leading ones of a head.  ``axes[i]`` (host integers; default 0) is
    the row of ``positions`` that turns pair i: a video token has time, height
    and width.  Pair i is components (2i, 2i+1) when ``interleaved``, otherwise
    (i, i + len(frequencies))."""

    def __init__(self, frequencies, axes=None, interleaved=False):
        device = _cuda_device("frequencies", frequencies)
        _check("frequencies", frequencies, 1, torch.float32, device)
        self.frequencies = frequencies
        self.interleaved = bool(interleaved)
        self.axes = 1
        self.pair_axis = None
        if axes is not None:
            axes = [int(x) for x in axes]
            _need(len(axes) == len(frequencies), f"axes: {len(frequencies)} pairs, {len(axes)} entries")
            _need(all(0 <= x < 16 for x in axes), "axes: entries must be 0..15")
            if any(axes):
                self.axes = max(axes) + 1
                self.pair_axis = torch.tensor(axes, dtype=torch.int32, device=device)
        self.components = 2 * self.frequencies.shape[0]
        self.device_index = device.index
        self.frequencies_ptr = frequencies.data_ptr()
        self.pair_axis_ptr = 0 if self.pair_axis is None else self.pair_axis.data_ptr()
        self._keep(self.frequencies, self.pair_axis)


def rotate_append(rotation, q, k, v, positions, slots, k_cache, v_cache, q_out=None, stream=None):
    """Rotated queries; rotated keys, and values, written to the cache in place.

    ``q`` [tokens, q_heads, dim], ``k`` and ``v`` [tokens, kv_heads, dim] (views
    of a joint projection are fine), all of one type with the cache: bfloat16,
    float16 or float32 (:func:`attention` reads the 16-bit ones of 64 or 128
    components).  ``positions`` int32 [tokens], or [axes, tokens] for a
    rotation of several axes.  ``slots`` int32 [tokens]: token ``s % page_size``
    of page ``s // page_size``; a slot outside the cache (-1, say) stores
    nothing; of two tokens with one slot, each component is one or the other's.
    ``q_out`` may be ``q`` itself.  Rotates in 32 bits, with angles
    formed in 64, and rounds once."""
    if not isinstance(q, torch.Tensor) or not q.is_cuda:
        raise ValueError("q: a CUDA tensor is wanted")
    dtype = q.dtype
    if dtype not in _DTYPES:
        raise ValueError(f"q: bfloat16, float16 or float32 is wanted, not {dtype}")
    if positions.ndim == 1:
        positions = positions[None]
    at = q.get_device()
    q_stride, k_stride, v_stride = q.stride(), k.stride(), v.stride()
    k_cache_stride, v_cache_stride, positions_stride, slots_stride = k_cache.stride(), v_cache.stride(), positions.stride(), slots.stride()
    if (len(q_stride) != 3 or len(k_stride) != 3 or len(v_stride) != 3 or len(k_cache_stride) != 4 or len(v_cache_stride) != 4
            or len(positions_stride) != 2 or slots_stride != (1,)
            or not (q_stride[2] == k_stride[2] == v_stride[2] == k_cache_stride[3] == v_cache_stride[3] == positions_stride[1] == 1)
            or not (dtype is k.dtype is v.dtype is k_cache.dtype is v_cache.dtype)
            or not (positions.dtype is slots.dtype is torch.int32)
            or not (at == k.get_device() == v.get_device() == k_cache.get_device() == v_cache.get_device()
                    == positions.get_device() == slots.get_device())):
        for name, t, ndim, kind in (("q", q, 3, dtype), ("k", k, 3, dtype), ("v", v, 3, dtype), ("k_cache", k_cache, 4, dtype),
                                    ("v_cache", v_cache, 4, dtype), ("positions", positions, 2, torch.int32),
                                    ("slots", slots, 1, torch.int32)):
            _check(name, t, ndim, kind, q.device)
    grads = _grads_on()
    if grads and (q.requires_grad or k.requires_grad or v.requires_grad or k_cache.requires_grad or v_cache.requires_grad
                  or rotation.frequencies.requires_grad):
        _no_backward()
    shape = q.shape
    tokens, q_heads, dim = shape
    cache_shape = k_cache.shape
    pages, page_size, kv_heads, cache_dim = cache_shape
    if v_cache.shape != cache_shape:
        raise ValueError("k_cache and v_cache have different shapes")
    if k.shape != (tokens, kv_heads, dim) or v.shape != k.shape or cache_dim != dim:
        raise ValueError("q, k, v and the caches do not fit together")
    axes, n = positions.shape
    if n != tokens or axes < rotation.axes:
        raise ValueError(f"positions: [{rotation.axes}, {tokens}] is wanted, not {list(positions.shape)}")
    if slots.shape[0] != tokens:
        raise ValueError(f"slots: {tokens} are wanted, not {slots.shape[0]}")
    if rotation.device_index != at:
        raise ValueError("rotation: on another device")
    if q_out is None:
        q_out = _empty_like(q, memory_format=_CONTIGUOUS) if stream is None else _new(stream, q, shape, dtype)
        q_out_stride = q_heads * dim, dim
    else:
        q_out_stride = _check("q_out", q_out, 3, dtype, q.device)[:2]
        if q_out.shape != shape:
            raise ValueError("q_out: another shape than q")
        if grads and q_out.requires_grad:
            _no_backward()
    try:
        a = _ROTATE_APPEND_ARGS.pack(
            _DTYPES[dtype], tokens, q_heads, kv_heads, dim, rotation.components, axes, rotation.interleaved, pages, page_size,
            q.data_ptr(), k.data_ptr(), v.data_ptr(), q_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            positions.data_ptr(), slots.data_ptr(), rotation.frequencies_ptr, rotation.pair_axis_ptr,
            q_stride[0], q_stride[1], k_stride[0], k_stride[1], v_stride[0], v_stride[1], q_out_stride[0], q_out_stride[1],
            k_cache_stride[0], k_cache_stride[1], k_cache_stride[2], v_cache_stride[0], v_cache_stride[1], v_cache_stride[2],
            positions_stride[0])
    except (struct.error, OverflowError) as e:
        raise _unfit(e) from None
    if stream is None:
        stream = _current_stream(at)
    if stream not in rotation._streams:
        rotation._used_on(stream)
    _call("emmy_rotate_append", at, stream, a)
    _written_to((k_cache, v_cache, q_out))
    return q_out


class AttentionPlan(_Kept):
    """How the attention of one batch is cut into units of work: made once from
    the host's lengths, used by every layer's call.

    Sequence s brings ``q_lens[s]`` new tokens to a cache that then holds
    ``kv_lens[s]`` of its tokens, the new ones last.  ``causal`` tokens see
    their own position and those before it, with a ``window`` only the last
    ``window`` of them; otherwise every token sees all ``kv_lens[s]``.
    ``q_heads`` is ``kv_heads`` times at most 128; ``head_dim`` is 64 or 128.
    ``ctas``: over how many CTAs the work is spread, one for each SM by default.
    Made by the host, in 30 us for one sequence, 140 to 300 for 64 to 256 that
    decode and 0.5 to 1.2 ms where chunks of hundreds of tokens are among them,
    and copied from pageable memory: the host waits for the current stream.

    A plan holds device memory (``words``, ``scratch``) that its calls write:
    they must not overlap on the GPU, so calls on several streams need a plan
    each.  It may be dropped while a call runs, on whichever stream, but not
    before a CUDA graph that holds its calls."""

    def __init__(self, q_lens, kv_lens, q_heads, kv_heads, head_dim, causal=True, window=None, device=None,
                 ctas=None):
        self._h = None
        q_lens, kv_lens = [int(x) for x in q_lens], [int(x) for x in kv_lens]
        _need(len(q_lens) == len(kv_lens), "q_lens and kv_lens have different lengths")
        _need(all(0 <= x <= 1 << 30 for x in q_lens + kv_lens), "lengths must be 0..2^30")
        _need(window is None or window >= 1, "window: at least 1, or None")
        _need(all(x is None or -1 << 31 <= x < 1 << 31 for x in (q_heads, kv_heads, head_dim, ctas)), "counts have to fit 32 bits")
        device = torch.device("cuda" if device is None else device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        if ctas is None:
            ctas = torch.cuda.get_device_properties(device).multi_processor_count
        n = len(q_lens)
        # (2^30: more than any length, and so no window)
        a = _PlanArgs(n, None, None, q_heads, kv_heads, head_dim, bool(causal), min(window or 0, 1 << 30), ctas)
        lens = (_i32 * (2 * n))(*q_lens, *kv_lens)
        a.q_lens, a.kv_lens = ctypes.addressof(lens), ctypes.addressof(lens) + 4 * n
        L = native.lib()
        h = ctypes.c_void_p()
        native.check(L.emmy_paged_plan_make(ctypes.byref(a), ctypes.byref(h)))
        self._h = h
        words, count, scratch = ctypes.c_void_p(), ctypes.c_size_t(), ctypes.c_size_t()
        native.check(L.emmy_paged_plan_data(h, ctypes.byref(words), ctypes.byref(count), ctypes.byref(scratch)))
        host = torch.frombuffer((_i32 * count.value).from_address(words.value), dtype=torch.int32)
        self.words = host.to(device, copy=True)
        self.scratch = torch.empty(scratch.value, dtype=torch.uint8, device=device)
        self.device, self.tokens, self.sequences = device, sum(q_lens), n
        self.q_heads, self.kv_heads, self.head_dim = int(q_heads), int(kv_heads), int(head_dim)
        self.shape = (self.tokens, self.q_heads, self.head_dim)
        self.scale = self.head_dim ** -0.5
        self.device_index = self.device.index
        self.words_ptr, self.scratch_ptr = self.words.data_ptr(), self.scratch.data_ptr()
        if device.type == "cuda":
            self._keep(self.words, self.scratch, own=True)

    def __del__(self):
        if self._h is not None:
            try:
                native.lib().emmy_paged_plan_free(self._h)
            except Exception:
                pass

    def check(self, stream=None):
        """Waits for the calls so far (with ``stream``, for those on it only) and raises
        if one of them gave up: its outputs are void, and later calls with this
        plan do nothing."""
        index = self.device.index
        if stream is None:
            stream = torch._C._cuda_getCurrentRawStream(index)
            if not self._streams <= {stream}:
                torch.cuda.synchronize(index)
        _call("emmy_paged_plan_status", index, stream, self._h, self.words.data_ptr())


def attention(plan, q, k_cache, v_cache, table, scale=None, out=None, lse=None, stream=None):
    """``(out, lse)``: softmax(scale q k^T) v of every new token over the keys
    that it sees, and the natural logarithm of the softmax's sum (float32
    [tokens, q_heads]; what joins attention over several parts of a cache).

    ``q`` [tokens, q_heads, head_dim], the sequences' tokens in order;
    bfloat16 or float16 like the cache.  ``table`` int32 [sequences, pages]:
    the pages of each sequence in order (entries after its last page are not
    read; a page outside the cache reads as zeros).  page_size is 8, 16, 32, 64
    or a multiple of 128.  ``scale`` defaults to 1/sqrt(head_dim).  A token
    that sees no key gets 0, and -inf; where none sees any, cache and table may
    be empty.  What lies in the cache beyond a
    sequence's length is never used, whatever it holds.  A key that is not finite
    concerns the tokens that see it; a value that some tokens of a chunk see and
    others do not must be finite.  An infinite value that all of them see makes
    its component infinite (NaN, where its weight rounds to 0 in the cache's
    type)."""
    if not isinstance(q, torch.Tensor) or not q.is_cuda:
        raise ValueError("q: a CUDA tensor is wanted")
    dtype = q.dtype
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError(f"q: bfloat16 or float16 is wanted, not {dtype}")
    at = q.get_device()
    q_stride, k_cache_stride, v_cache_stride, table_stride = q.stride(), k_cache.stride(), v_cache.stride(), table.stride()
    if (len(q_stride) != 3 or len(k_cache_stride) != 4 or len(v_cache_stride) != 4 or len(table_stride) != 2
            or not (q_stride[2] == k_cache_stride[3] == v_cache_stride[3] == table_stride[1] == 1)
            or not (dtype is k_cache.dtype is v_cache.dtype) or table.dtype is not torch.int32
            or not (at == k_cache.get_device() == v_cache.get_device() == table.get_device())):
        for name, t, ndim, kind in (("q", q, 3, dtype), ("k_cache", k_cache, 4, dtype), ("v_cache", v_cache, 4, dtype),
                                    ("table", table, 2, torch.int32)):
            _check(name, t, ndim, kind, q.device)
    grads = _grads_on()
    if grads and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        _no_backward()
    if at != plan.device_index:
        raise ValueError(f"q: on {q.device}, the plan on {plan.device}")
    shape = plan.shape
    if q.shape != shape:
        raise ValueError(f"q: the plan is for {list(shape)}, not {list(q.shape)}")
    cache_shape = k_cache.shape
    if v_cache.shape != cache_shape:
        raise ValueError("k_cache and v_cache have different shapes")
    pages, page_size, kv_heads, dim = cache_shape
    if kv_heads != plan.kv_heads or dim != plan.head_dim:
        raise ValueError(f"k_cache: the plan is for {plan.kv_heads} heads of {plan.head_dim}, not {kv_heads} of {dim}")
    rows, width = table.shape
    if rows != plan.sequences:
        raise ValueError(f"table: {plan.sequences} rows are wanted, not {rows}")
    given = out is not None or lse is not None
    if out is None:
        out = _empty_like(q, memory_format=_CONTIGUOUS) if stream is None else _new(stream, q, shape, dtype)
        out_stride = shape[1] * dim, dim
    else:
        out_stride = _check("out", out, 3, dtype, q.device)[:2]
        if out.shape != shape:
            raise ValueError("out: another shape than q")
        if grads and out.requires_grad:
            _no_backward()
    if lse is None:
        lse = q.new_empty(shape[:2], dtype=torch.float32) if stream is None else _new(stream, q, shape[:2], torch.float32)
    else:
        _check("lse", lse, 2, torch.float32, q.device)
        if lse.shape != shape[:2] or not lse.is_contiguous():
            raise ValueError(f"lse: contiguous {list(shape[:2])} is wanted")
        if grads and lse.requires_grad:
            _no_backward()
    try:
        a = _ATTENTION_ARGS.pack(
            _DTYPES[dtype], pages, page_size, width, plan.scale if scale is None else scale,
            q.data_ptr(), out.data_ptr(), lse.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), table.data_ptr(),
            plan.words_ptr, plan.scratch_ptr, q_stride[0], q_stride[1], out_stride[0], out_stride[1],
            k_cache_stride[0], k_cache_stride[1], k_cache_stride[2], v_cache_stride[0], v_cache_stride[1], v_cache_stride[2],
            table_stride[0])
    except (struct.error, OverflowError) as e:
        raise _unfit(e) from None
    if stream is None:
        stream = _current_stream(at)
    if stream not in plan._streams:
        plan._used_on(stream)
    _call("emmy_paged_attention", at, stream, plan._h, a)
    if given:
        _written_to((out, lse))
    return out, lse
