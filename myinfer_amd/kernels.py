"""Typed wrappers around libkvq.so's entry points (torch tensors in, torch tensors out).

Every wrapper validates shapes on the host, passes raw pointers and strides through the C ABI
and launches on the tensors' current HIP stream. Scratch memory (the attention workspace) is a
zero-filled torch allocation cached per (device, stream); the library itself allocates nothing.
"""

from __future__ import annotations

import contextlib
import ctypes
import functools
import weakref
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import torch

from . import _lib

Triple = Tuple[torch.Tensor, torch.Tensor, torch.Tensor]

_workspaces: dict = {}


def new_workspace(nbytes: int, device) -> torch.Tensor:
    """A zero-filled attention workspace. The kernels keep their split counters in it and leave
    them at zero after every call, so a workspace is zeroed once, when it is allocated."""
    return torch.zeros(max(int(nbytes), 1 << 20), dtype=torch.uint8, device=device)


def _workspace(device: torch.device, stream: int, nbytes: int) -> torch.Tensor:
    key = (device.index, stream)
    buf = _workspaces.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = new_workspace(nbytes, device)
        _workspaces[key] = buf
    return buf


def _require_cuda(*tensors: torch.Tensor) -> torch.device:
    dev = tensors[0].device
    if dev.type != "cuda":
        raise ValueError(f"libkvq operates on GPU tensors; got a tensor on {dev}")
    for t in tensors[1:]:
        if t.device != dev:
            raise ValueError(f"all tensors must be on {dev}; got {t.device}")
    return dev


def _on_device(dev: torch.device):
    """A context in which `dev` is the current device (launches go to streams of the current one)."""
    if dev.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


def _native(t) -> tuple:
    """(the native host path, the raw current stream) for a tensor on the current GPU, else (None, 0). What its functions
    answer: the result, None (the Python path serves or refuses the call), or a failed launch's status."""
    dev = t.get_device() if torch.is_tensor(t) else -1
    if dev < 0 or dev != torch._C._cuda_getDevice():
        return None, 0
    return _lib.host(), torch._C._cuda_getCurrentRawStream(dev)


def _check_triple(tr: Sequence[torch.Tensor], name: str) -> None:
    if len(tr) != 3:
        raise ValueError(f"{name} must be a (codes, scales, biases) triple")


# ---- range exponents (include/kvq.h, kvq_qtensor.range_exp)
#
# A quantized cache keeps one int32 in device memory, its range exponent E: the appends raise it to
# the smallest E >= 0 with every dequantized value within 2^15 * 2^E, and the quantized prefill
# kernels stage their fp16 operands times 2^-E, so a bf16 cache whose values leave the fp16 range
# still gives finite results. The word belongs to the cache's buffers: it is registered here under
# the storage of the codes buffer, and every call that is handed a view of those buffers (the
# reference-style entry points pass only the (codes, scales, biases) views) finds it again.

_range_words: dict = {}  # codes storage address -> (weak reference to the codes buffer, int32 word)


def register_range_word(codes: torch.Tensor, word: torch.Tensor) -> None:
    """Attach a cache's range word (a one-element int32 tensor on the codes' device) to the codes
    buffer: appends into views of it raise the word, attention over views of it reads it."""
    if word.dtype != torch.int32 or word.numel() != 1 or word.device != codes.device:
        raise ValueError("a range word is a one-element int32 tensor on the cache's device")
    key = codes.untyped_storage().data_ptr()
    if len(_range_words) > 4096:  # drop entries whose buffers are gone
        for k in [k for k, (ref, _) in _range_words.items() if ref() is None]:
            del _range_words[k]
    _range_words[key] = (weakref.ref(codes), word)


def range_word(codes: torch.Tensor) -> Optional[torch.Tensor]:
    """The range word registered for the buffer `codes` is a view of, or None."""
    hit = _range_words.get(codes.untyped_storage().data_ptr())
    if hit is None:
        return None
    buf = hit[0]()
    if buf is None or buf.untyped_storage().data_ptr() != codes.untyped_storage().data_ptr():
        return None
    return hit[1]


def range_exponent(triple: Triple, bits: int) -> torch.Tensor:
    """The range exponent of a (codes, scales, biases) triple computed from its scales and biases on
    its device (no host synchronization): the smallest E >= 0 with max(|b|, |b + (2^bits - 1) s|)
    <= 2^15 * 2^E over every group, as a one-element int32 tensor. For triples that carry no
    registered word."""
    _, scales, biases = triple
    s, b = scales.float(), biases.float()
    if s.numel() == 0:
        return torch.zeros(1, dtype=torch.int32, device=scales.device)
    top = b + float((1 << bits) - 1) * s
    bound = torch.nan_to_num(torch.maximum(b.abs(), top.abs()), nan=0.0, posinf=float("inf")).amax()
    e = torch.ceil(torch.log2(bound * (1.0 / 32768.0)))
    e = torch.nan_to_num(e, nan=127.0, posinf=127.0, neginf=0.0).clamp(0.0, 127.0)
    return e.to(torch.int32).reshape(1)


@dataclass(frozen=True)
class Rope:
    """Rotary position embedding as mlx's nn.RoPE(dims, traditional, base, scale) applies it: row l
    of a call at position offset + l, pair i turned by (position * scale) * base^(-2i/dims)."""

    dims: int
    traditional: bool = False
    base: float = 10000.0
    scale: float = 1.0

    def params(self, offset: int) -> "_lib.RopeParams":
        return _lib.RopeParams(int(self.dims), int(bool(self.traditional)), float(self.base), float(self.scale),
                               int(offset))


def rope(x: torch.Tensor, r: Rope, offset: int = 0) -> torch.Tensor:
    """Rotate x [B, H, L, D] (float16/bfloat16, CUDA) in place, rows at positions offset + l, and
    return it: the query side of a fused RoPE + cache update (kernels.metal:106-160)."""
    dev = _require_cuda(x)
    if x.dim() != 4:
        raise ValueError(f"x must be [B, H, L, D], got {tuple(x.shape)}")
    B, H, L, D = x.shape
    xr, rp = _lib.rows(x), r.params(offset)
    rc = _lib.lib().kvq_rope(ctypes.byref(xr), ctypes.byref(rp), B, H, L, D, _lib.dtype_code(x.dtype),
                             _lib.stream_ptr(dev))
    _lib.check(rc, "kvq_rope")
    return x


@dataclass(frozen=True)
class RopeAxes:
    """Rotary position embedding at positions given per row, over 1 to 4 axes: the time, height and width of an
    image's or a video's tokens, or one axis for rows that are not consecutive (a tree of drafted tokens). Pair i
    of a row turns by position[axis(i)] * scale * freq(i).

    ``sections``: pairs of each axis, dims / 2 in all (default: one axis). ``interleaved``: False: the first
    sections[0] pairs belong to axis 0, the next sections[1] to axis 1, ...; True: pairs are dealt to the axes in turn,
    passing over those that have all of theirs. ``restart``: False: freq(i) = base^(-2 i / dims); True: every axis
    counts its own pairs, base^(-j / sections[axis]) for its pair j. ``traditional`` as in Rope.

    Angles are formed and reduced in double precision (Rope's in fp32, as mlx's are: the two agree to an ulp of the
    rows' type at near positions, and part at far ones)."""

    dims: int
    sections: Tuple[int, ...] = ()
    traditional: bool = False
    base: float = 10000.0
    scale: float = 1.0
    interleaved: bool = False
    restart: bool = False

    def __post_init__(self):
        sections = tuple(int(n) for n in self.sections) or (int(self.dims) // 2,)
        if not 1 <= len(sections) <= _lib.MAX_AXES:
            raise ValueError(f"1 to {_lib.MAX_AXES} axes, got sections {sections}")
        if min(sections) < 1 or sum(sections) != int(self.dims) // 2:
            raise ValueError(f"sections {sections} must be at least 1 each and dims / 2 = {int(self.dims) // 2} in all")
        object.__setattr__(self, "sections", sections)

    @property
    def axes(self) -> int:
        return len(self.sections)

    def params(self) -> "_lib.Axes":
        """The descriptor without positions (``set_positions``)."""
        return _lib.Axes(int(self.dims), int(bool(self.traditional)), self.axes, (ctypes.c_int * _lib.MAX_AXES)(*self.sections),
                         int(bool(self.interleaved)), int(bool(self.restart)), float(self.base), float(self.scale), None, 0, 0, 0)


def _set_positions(desc: "_lib.Axes", positions: torch.Tensor, B: int, L: int, dev: torch.device) -> None:
    """Point `desc` at int32 positions [axes, B, L] (or [axes, L], the same for every sequence) after their checks."""
    A = desc.axes
    if not torch.is_tensor(positions) or positions.dtype != torch.int32 or positions.device != dev:
        raise ValueError(f"positions must be an int32 tensor on {dev}")
    if tuple(positions.shape) == (A, B, L):
        sa, sb, sl = positions.stride()
    elif tuple(positions.shape) == (A, L):
        (sa, sl), sb = positions.stride(), 0
    else:
        raise ValueError(f"positions must be [axes, B, L] = {(A, B, L)} or [axes, L], got {tuple(positions.shape)}")
    desc.positions, desc.pos_stride_a, desc.pos_stride_b, desc.pos_stride_l = positions.data_ptr(), sa, sb, sl


_axes_desc = functools.lru_cache(maxsize=64)(RopeAxes.params)


def rope_axes(x: torch.Tensor, r: RopeAxes, positions: torch.Tensor) -> torch.Tensor:
    """Rotate x [B, H, L, D] (float16/bfloat16, CUDA) in place, row l of sequence b at positions[:, b, l], and return
    it. positions: int32 [axes, B, L] or [axes, L]. A broadcast x, whose rows share their memory, is refused."""
    host, stream = _native(x)
    if host is not None:
        desc = _axes_desc(r)
        done = host.rope_axes(ctypes.addressof(desc), x, positions, stream)
        if done is True:
            return x
        if done is not None:
            _lib.check(done, "kvq_rope_axes")
    dev = _require_cuda(x)
    if x.dim() != 4:
        raise ValueError(f"x must be [B, H, L, D], got {tuple(x.shape)}")
    B, H, L, D = x.shape
    xr, rp = _lib.rows(x), r.params()
    _set_positions(rp, positions, B, L, dev)
    if x.numel() == 0:
        return x
    with _on_device(dev):
        rc = _lib.lib().kvq_rope_axes(ctypes.byref(xr), ctypes.byref(rp), B, H, L, D, _lib.dtype_code(x.dtype),
                                      _lib.stream_ptr(dev))
    _lib.check(rc, "kvq_rope_axes")
    return x


class AxesAppendCall:
    """A quantize-append into fixed destination buffers, or with ``paged`` into the pages of fixed pools, with the rotation
    of the step's keys and queries at given positions, its descriptors built once (``prepare_axes_append``). Launches on the
    stream current at the call."""

    def __init__(self, k_dst: Triple, v_dst: Optional[Triple], rope: RopeAxes, group_size: int, bits: int):
        _check_triple(k_dst, "k_dst")
        tens = list(k_dst)
        if v_dst is not None:
            _check_triple(v_dst, "v_dst")
            tens += list(v_dst)
            if any(tuple(a.shape) != tuple(b.shape) for a, b in zip(k_dst, v_dst)) or v_dst[1].dtype != k_dst[1].dtype:
                raise ValueError("k_dst and v_dst must have the same shapes and dtype")
        self._dev = _require_cuda(*tens)
        # (the range words are held too: the descriptors point to them)
        self._keep = (k_dst, v_dst, range_word(k_dst[0]), None if v_dst is None else range_word(v_dst[0]))
        codes, scales, _ = k_dst
        if tuple(scales.shape[:3]) != tuple(codes.shape[:3]):
            raise ValueError("the destination's codes and scales must have the same rows")
        self._lead, self._rows = tuple(codes.shape[:2]), codes.shape[2]
        self._widths = (codes.shape[3], scales.shape[3])
        self._kq = _lib.qtensor(*k_dst, range_exp=range_word(k_dst[0]))
        self._vq = None if v_dst is None else _lib.qtensor(*v_dst, range_exp=range_word(v_dst[0]))
        self._dtype, self._code = scales.dtype, _lib.dtype_code(scales.dtype)
        self._bits, self._group = int(bits), int(group_size)
        self.rope = rope
        self._rp = rope.params()
        self._state = _lib.AppendState(
            None, ctypes.addressof(self._kq), None if self._vq is None else ctypes.addressof(self._vq),
            ctypes.addressof(self._rp), *self._lead, self._rows, *self._widths, self._bits, self._group, self._code,
            self._dev.index, None)
        self._state_ptr = ctypes.addressof(self._state)

    def _check(self, k, v, positions, queries) -> tuple:
        if k.dtype != self._dtype or k.device != self._dev or k.dim() != 4:
            raise ValueError(f"keys must be {self._dtype} [B, H, L, D] on {self._dev}")
        B, H, L, D = k.shape
        if self._widths != (D * self._bits // 32, D // self._group):
            raise ValueError("destination row widths do not match D, bits and group_size")
        if (v is None) != (self._vq is None) or (v is not None and (v.shape != k.shape or v.dtype != k.dtype or
                                                                    v.device != self._dev)):
            raise ValueError("values must match the keys and a value destination")
        if queries is not None and (queries.dtype != k.dtype or queries.device != self._dev or queries.dim() != 4 or
                                    queries.shape[0] != B or tuple(queries.shape[2:]) != (L, D)):
            raise ValueError(f"queries must be {self._dtype} [{B}, Hq, {L}, {D}] on {self._dev}")
        rp = _lib.Axes.from_buffer_copy(self._rp)
        _set_positions(rp, positions, B, L, self._dev)
        return rp, B, H, L, D

    def _launch(self, k, v, queries, rp, B, H, L, D, row_offset, paging) -> None:
        if k.numel() == 0:
            return
        if queries is not None and queries.numel() == 0:
            queries = None
        kr = _lib.rows(k)
        vr = None if v is None else _lib.rows(v)
        qr = None if queries is None else _lib.rows(queries)
        ref = ctypes.byref
        with _on_device(self._dev):
            rc = _lib.lib().kvq_rope_axes_append(
                ref(kr), ref(self._kq), None if vr is None else ref(vr), None if vr is None else ref(self._vq),
                None if qr is None else ref(qr), 0 if qr is None else queries.shape[1], ref(rp), *paging, int(row_offset), B, H,
                L, D, self._bits, self._group, self._code, _lib.stream_ptr(self._dev))
        _lib.check(rc, "kvq_rope_axes_append")

    def __call__(self, k: torch.Tensor, v: Optional[torch.Tensor], positions: torch.Tensor, row_offset: int,
                 queries: Optional[torch.Tensor] = None) -> None:
        if self._native_append(k, v, positions, row_offset, queries, None, None):
            return
        rp, B, H, L, D = self._check(k, v, positions, queries)
        if (B, H) != self._lead:
            raise ValueError(f"destination leads {self._lead} do not match source {(B, H)}")
        if row_offset < 0 or row_offset + L > self._rows:
            raise ValueError(f"rows [{row_offset}, {row_offset + L}) exceed the destination's {self._rows} rows")
        self._launch(k, v, queries, rp, B, H, L, D, row_offset, (0, None, 0, None))

    def paged(self, k: torch.Tensor, v: Optional[torch.Tensor], positions: torch.Tensor, block_tables: torch.Tensor,
              starts: Optional[torch.Tensor] = None, row_offset: int = 0, queries: Optional[torch.Tensor] = None) -> None:
        """``paged_rope_axes_append`` into the prepared pools."""
        if self._native_append(k, v, positions, row_offset, queries, block_tables, starts):
            return
        rp, B, H, L, D = self._check(k, v, positions, queries)
        if self._lead[1] != H or self._rows != PAGE_ROWS:
            raise ValueError(f"pools must be [num_pages, {H}, {PAGE_ROWS}, *]")
        block_tables = _whole_table(block_tables, B, self._dev)
        self._launch(k, v, queries, rp, B, H, L, D, row_offset,
                     (self._lead[0], block_tables.data_ptr(), block_tables.stride(0), _check_starts(starts, B, self._dev)))

    def _native_append(self, k, v, positions, row_offset, queries, table, starts) -> bool:
        host, stream = _native(k)
        if host is None:
            return False
        done = host.axes_append(self._state_ptr, k, v, positions, row_offset, queries, stream, table, starts)
        if done is not None and done is not True:
            _lib.check(done, "kvq_rope_axes_append")
        return done is True


def prepare_axes_append(k_dst: Triple, v_dst: Optional[Triple] = None, *, rope: RopeAxes, group_size: int = 64,
                        bits: int = 8) -> AxesAppendCall:
    """Build an ``AxesAppendCall`` for repeated appends into the same (codes, scales, biases) buffers."""
    return AxesAppendCall(k_dst, v_dst, rope, group_size, bits)


def quantize_append(k: torch.Tensor, k_dst: Triple, v: Optional[torch.Tensor] = None, v_dst: Optional[Triple] = None,
                    row_offset: int = 0, group_size: int = 64, bits: int = 8, rope: Optional[Rope] = None,
                    rope_offset: Optional[int] = None) -> None:
    """Quantize k (and v) [B, H, L, D] and store them at rows [row_offset, row_offset + L) of the
    (codes, scales, biases) buffers k_dst (and v_dst), in one kernel launch. With `rope`, the keys
    are rotated first (row l at position rope_offset + l, rope_offset defaulting to row_offset) and
    rounded to their dtype before they are quantized; k itself is not modified."""
    _check_triple(k_dst, "k_dst")
    tens = [k, *k_dst]
    if v is not None:
        if v_dst is None:
            raise ValueError("v_dst is required with v")
        _check_triple(v_dst, "v_dst")
        if v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError("k and v must have the same shape and dtype")
        tens += [v, *v_dst]
    dev = _require_cuda(*tens)
    B, H, L, D = k.shape
    for tr in [k_dst] + ([v_dst] if v is not None else []):
        codes, scales, _ = tr
        if codes.shape[:2] != (B, H) or scales.shape[:2] != (B, H):
            raise ValueError(f"destination leads {tuple(codes.shape[:2])} do not match source {(B, H)}")
        if row_offset + L > codes.shape[2] or row_offset + L > scales.shape[2]:
            raise ValueError(f"rows [{row_offset}, {row_offset + L}) exceed the destination's {codes.shape[2]} rows")
        if codes.shape[3] != D * bits // 32 or scales.shape[3] != D // group_size:
            raise ValueError("destination row widths do not match D, bits and group_size")
        if scales.dtype != k.dtype:
            raise ValueError("scales/biases must have the dtype of the rows (MLX stores them in T)")
    L_ = _lib.lib()
    kr, kq = _lib.rows(k), _lib.qtensor(*k_dst, range_exp=range_word(k_dst[0]))
    if v is not None:
        vr, vq = _lib.rows(v), _lib.qtensor(*v_dst, range_exp=range_word(v_dst[0]))
        vr_p, vq_p = ctypes.byref(vr), ctypes.byref(vq)
    else:
        vr_p = vq_p = None
    if rope is None:
        rc = L_.kvq_quantize_append(ctypes.byref(kr), ctypes.byref(kq), vr_p, vq_p, int(row_offset), B, H, L, D,
                                    int(bits), int(group_size), _lib.dtype_code(k.dtype), _lib.stream_ptr(dev))
        _lib.check(rc, "kvq_quantize_append")
    else:
        rp = rope.params(row_offset if rope_offset is None else rope_offset)
        rc = L_.kvq_rope_quantize_append(ctypes.byref(kr), ctypes.byref(kq), vr_p, vq_p, ctypes.byref(rp),
                                         int(row_offset), B, H, L, D, int(bits), int(group_size),
                                         _lib.dtype_code(k.dtype), _lib.stream_ptr(dev))
        _lib.check(rc, "kvq_rope_quantize_append")


class AppendCall:
    """A quantize-append into fixed destination buffers with its C-ABI descriptors built once.

    ``prepare_append`` validates the destinations; calling the object with new source rows fills
    two preallocated row descriptors and makes one foreign call, so a decode loop pays a few
    microseconds of host time per layer instead of rebuilding every descriptor. Launches go to
    the stream that was current at preparation time.
    """

    def __init__(self, k_dst: Triple, v_dst: Optional[Triple], group_size: int, bits: int,
                 rope: Optional[Rope]):
        _check_triple(k_dst, "k_dst")
        tens = list(k_dst)
        if v_dst is not None:
            _check_triple(v_dst, "v_dst")
            tens += list(v_dst)
        self._dev = _require_cuda(*tens)
        self._k_dst, self._v_dst = k_dst, v_dst  # the descriptors point into these
        codes, scales, _ = k_dst
        self._lead = tuple(codes.shape[:2])
        self._rows = min(codes.shape[2], scales.shape[2])
        self._widths = (codes.shape[3], scales.shape[3])
        if v_dst is not None:
            if tuple(v_dst[0].shape) != tuple(codes.shape) or tuple(v_dst[1].shape) != tuple(scales.shape):
                raise ValueError("k_dst and v_dst must have the same shapes")
            if v_dst[1].dtype != scales.dtype:
                raise ValueError("k_dst and v_dst must share a dtype")
        self._kq = _lib.qtensor(*k_dst, range_exp=range_word(k_dst[0]))
        self._vq = _lib.qtensor(*v_dst, range_exp=range_word(v_dst[0])) if v_dst is not None else None
        self._kr, self._vr = _lib.Rows(), _lib.Rows()
        self._dtype = k_dst[1].dtype
        self._code = _lib.dtype_code(self._dtype)
        self._bits, self._group = int(bits), int(group_size)
        self._rope = rope
        self._rp = rope.params(0) if rope is not None else None
        lib = _lib.lib()
        self._fn = lib.kvq_rope_quantize_append if rope is not None else lib.kvq_quantize_append
        self._stream = _lib.stream_ptr(self._dev)
        self._symbol = "kvq_rope_quantize_append" if rope is not None else "kvq_quantize_append"
        self._host = _lib.host().append
        self._state = _lib.AppendState(
            ctypes.cast(self._fn, ctypes.c_void_p).value, ctypes.addressof(self._kq),
            None if self._vq is None else ctypes.addressof(self._vq),
            None if self._rp is None else ctypes.addressof(self._rp), *self._lead, self._rows, *self._widths, self._bits,
            self._group, self._code, self._dev.index, self._stream)
        self._state_ptr = ctypes.addressof(self._state)

    def __call__(self, k: torch.Tensor, v: Optional[torch.Tensor], row_offset: int,
                 rope_offset: Optional[int] = None) -> None:
        # the native host path; anything it does not take is checked, served or refused below
        done = self._host(self._state_ptr, k, v, row_offset, row_offset if rope_offset is None else rope_offset)
        if done is True:
            return
        if done is not None:  # a failed launch, which is not tried again
            _lib.check(done, self._symbol)
        if k.dtype != self._dtype or k.device != self._dev or k.dim() != 4 or k.stride(-1) != 1:
            raise ValueError("rows must match the prepared dtype and device, as [B, H, L, D] with D contiguous")
        B, H, L, D = k.shape
        if (B, H) != self._lead:
            raise ValueError(f"destination leads {self._lead} do not match source {(B, H)}")
        if row_offset < 0 or row_offset + L > self._rows:
            raise ValueError(f"rows [{row_offset}, {row_offset + L}) exceed the destination's {self._rows} rows")
        if self._widths != (D * self._bits // 32, D // self._group):
            raise ValueError("destination row widths do not match D, bits and group_size")
        kr = self._kr
        kr.data = k.data_ptr()
        kr.stride_b, kr.stride_h, kr.stride_l = k.stride()[:3]
        vr_p = vq_p = None
        if v is not None:
            if self._vq is None or v.shape != k.shape or v.dtype != k.dtype or v.stride(-1) != 1:
                raise ValueError("values must match the keys and a prepared value destination")
            vr = self._vr
            vr.data = v.data_ptr()
            vr.stride_b, vr.stride_h, vr.stride_l = v.stride()[:3]
            vr_p, vq_p = ctypes.byref(vr), ctypes.byref(self._vq)
        if self._rp is None:
            rc = self._fn(ctypes.byref(kr), ctypes.byref(self._kq), vr_p, vq_p, int(row_offset), B, H, L, D,
                          self._bits, self._group, self._code, self._stream)
        else:
            self._rp.offset = int(row_offset if rope_offset is None else rope_offset)
            rc = self._fn(ctypes.byref(kr), ctypes.byref(self._kq), vr_p, vq_p, ctypes.byref(self._rp),
                          int(row_offset), B, H, L, D, self._bits, self._group, self._code, self._stream)
        if rc:
            _lib.check(rc, self._symbol)


def prepare_append(k_dst: Triple, v_dst: Optional[Triple] = None, *, group_size: int = 64, bits: int = 8,
                   rope: Optional[Rope] = None) -> AppendCall:
    """Build an ``AppendCall`` for repeated appends into the same (codes, scales, biases) buffers."""
    return AppendCall(k_dst, v_dst, group_size, bits, rope)


def quantize(x: torch.Tensor, group_size: int = 64, bits: int = 8) -> Triple:
    """Counterpart of mx.quantize(x, group_size, bits) for x [..., D] on the GPU:
    returns (codes uint32 [..., D*bits/32], scales [..., D/G], biases [..., D/G])."""
    _require_cuda(x)
    lead = x.shape[:-1]
    D = x.shape[-1]
    x4 = x.reshape(1, 1, -1, D)
    if x4.stride(-1) != 1:
        x4 = x4.contiguous()
    n = x4.shape[2]
    codes = torch.empty((1, 1, n, D * bits // 32), dtype=torch.uint32, device=x.device)
    scales = torch.empty((1, 1, n, D // group_size), dtype=x.dtype, device=x.device)
    biases = torch.empty_like(scales)
    quantize_append(x4, (codes, scales, biases), row_offset=0, group_size=group_size, bits=bits)
    return (codes.reshape(*lead, -1), scales.reshape(*lead, -1), biases.reshape(*lead, -1))


def _check_read(k: Triple, v: Optional[Triple], group_size: int, bits: int):
    """The device, leading dims and head dim of triples to be read back, after their checks."""
    tens = []
    for name, tr in (("keys", k), ("values", v)):
        if tr is None:
            continue
        _check_triple(tr, name)
        if any(x.dim() != 4 for x in tr) or tr[1].shape[:3] != tr[0].shape[:3]:
            raise ValueError(f"{name} must be 4-D (codes, scales, biases) with the same rows")
        if tr[0].shape[3] * 32 // bits != tr[1].shape[3] * group_size:
            raise ValueError(f"{name}: codes of {tr[0].shape[3]} words and {tr[1].shape[3]} groups are not rows of one "
                             f"width at {bits} bits and group_size {group_size}")
        if tuple(tr[0].shape) != tuple(k[0].shape) or tr[1].dtype != k[1].dtype:
            raise ValueError("keys and values must have the same shapes and dtype")
        tens += list(tr)
    return _require_cuda(*tens), tuple(k[0].shape[:3]), k[1].shape[3] * group_size


def _read_out(out, n: int, shape, dtype, dev, fresh):
    if out is None:
        return tuple(fresh(shape, dtype=dtype, device=dev) for _ in range(n))
    out = tuple(out)
    if len(out) != n or any(tuple(o.shape) != shape or o.dtype != dtype or o.device != dev for o in out):
        raise ValueError(f"out must be {n} {dtype} tensors of shape {shape} on {dev}")
    return out


def read_rows(k: Triple, v: Triple, start: int, stop: int, *, group_size: int = 64, bits: int = 8, out=None, table=None,
              seq_lens=None):
    """Rows [start, stop) of K and V triples through the native host path, as ``dequantize_rows`` of those rows or, with a
    block table, ``paged_dequantize`` into `out`; None for a call it does not take."""
    host, stream = _native(k[1])
    if host is None:
        return None
    got = host.dequantize(k, v, start, stop, group_size, bits, out, table, seq_lens, stream)
    if type(got) is int:
        _lib.check(got, "kvq_dequantize" if table is None else "kvq_paged_dequantize")
    return got


def dequantize_rows(k: Triple, v: Optional[Triple] = None, *, group_size: int = 64, bits: int = 8, out=None):
    """The rows of quantized triples [B, H, S, *] (views of a cache) as values [B, H, S, D] in their dtype, K and V in
    one launch: (K, V), or (K,) without v. `out`: the tensors to fill instead of new ones."""
    if v is not None and type(k) is tuple and len(k) == 3 and k[0].dim() == 4:
        got = read_rows(k, v, 0, k[0].shape[2], group_size=group_size, bits=bits, out=None if out is None else tuple(out))
        if got is not None:
            return got
    dev, (B, H, S), D = _check_read(k, v, group_size, bits)
    outs = _read_out(out, 1 if v is None else 2, (B, H, S, D), k[1].dtype, dev, torch.empty)
    if outs[0].numel() == 0:
        return outs
    kq, kr = _lib.qtensor(*k), _lib.rows(outs[0])
    vq, vr = (None, None) if v is None else (_lib.qtensor(*v), _lib.rows(outs[1]))
    ref = ctypes.byref
    with _on_device(dev):
        rc = _lib.lib().kvq_dequantize(ref(kq), ref(kr), None if v is None else ref(vq), None if v is None else ref(vr), 0, B, H,
                                       S, D, int(bits), int(group_size), _lib.dtype_code(k[1].dtype), _lib.stream_ptr(dev))
    _lib.check(rc, "kvq_dequantize")
    return outs


def dequantize(codes: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, group_size: int = 64,
               bits: int = 8) -> torch.Tensor:
    """Counterpart of mx.dequantize(w, scales, biases, group_size, bits) on the GPU: codes uint32 [..., D*bits/32],
    scales and biases [..., D/G] -> values [..., D] in the scales' dtype."""
    if codes.shape[:-1] != scales.shape[:-1]:
        raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} have different leading dims")
    lead = codes.shape[:-1]
    flat = [x.reshape(1, 1, -1, x.shape[-1]).contiguous() for x in (codes, scales, biases)]
    return dequantize_rows(tuple(flat), group_size=group_size, bits=bits)[0].reshape(*lead, -1)


FP16_MAX = 65504.0


def fits_fp16_operands(triple: Triple, bits: int) -> bool:
    """Whether every dequantized value s * c + b (c in [0, 2^bits - 1]) of a (codes, scales,
    biases) triple lies inside the fp16 range. The prefill kernel's dequantized operands are fp16:
    for a bf16 cache with a group outside that range its query rows come back NaN (decode is exact
    either way), so a caller whose bf16 K/V can exceed 65504 checks its cache once with this and
    routes those layers through decode. Works on the triple's device; returns a Python bool (a
    synchronisation on the GPU)."""
    _check_triple(triple, "triple")
    _, scales, biases = triple
    s, b = scales.float(), biases.float()
    hi = b + s * float((1 << bits) - 1)
    worst = torch.maximum(b.abs(), hi.abs())
    return bool(torch.isfinite(worst).all().item()) and bool((worst <= FP16_MAX).all().item())


NATIVE_HEAD_DIMS = (64, 128, 256)


def kernel_dim(D: int) -> int:
    """The width the kernels compute head dimension D at: 64, 128 or 256. Other multiples of 8 (up to
    256 for quantized caches, 128 for unquantized ones) run the decode kernel at the next width, with
    zero queries past their last dim, for every query length (quantized 96 up to 64 rows: past them
    the prefill kernel has a 96-wide form)."""
    return 64 if D <= 64 else 128 if D <= 128 else 256


def decode_rows_per_pass(D: int, group_size: int = 64) -> int:
    """Query rows (heads of a GQA group x query positions) one decode pass serves: the 16 MFMA
    columns hold each row once per scale group of the kernel's width (an unquantized cache counts as
    group 64)."""
    return 16 * group_size // kernel_dim(D)


def _auto_kernel(rep_rows: int, D: int, group_size: int, *, dense: bool, units: int, keys: int) -> str:
    """Decode or prefill for `units` (sequence, KV head) pairs of `rep_rows` query rows over `keys` keys.

    Decode while a KV head's rows fit at most two decode passes over its keys (one pass for group 64,
    where 8 rows fit one pass). Past that, over quantized caches and below the rows of one prefill
    workgroup (256, or 128 at 256 dims), the kernel that is faster: a decode call's time grows with its
    passes (about 25 us per 2^20 passes x units x keys at 128 dims), a prefill kernel's is that of the
    whole row block and of merging the splits that a few such blocks are cut into. Measured at 128 dims,
    8 bits, decode against prefill in us:
      4 units, 8192 keys: 14.4 / 18.4 at 64 rows, 20.1 / 19.9 at 128; 2048 keys: 13.4 / 18.2 at 192;
      16 units, 32768 keys: 57 / 72 at 32 rows, 105 / 72 at 48; 32 units, 32768 keys: 110 / 131 at 32;
      prompts, where causality halves the prefill kernel's work: 32 units 7.8 / 11.6 at 128 tokens (512
      row blocks, the last that run at once), 15.1 / 16.8 at 200, 25.5 / 18.2 at 330;
    at 256 dims (4 rows a pass) 22 / 24 at 16 rows, 28 / 24 at 24 (8 units, 8192 keys), 57 / 59 at 16
    rows of 32768 keys. Unquantized caches keep to one pass.

    Head dims 64, 128 and 256 have prefill kernels; the others run the decode kernel at every length,
    but for quantized caches of 96 dims (groups of 32), which have one past 64 rows. At head_dim 256 the
    unquantized entry points run the head_dim-256 kernel for every query length."""
    if D == 96 and not dense:
        return "decode" if rep_rows <= 64 else "prefill"
    if D not in NATIVE_HEAD_DIMS:
        return "decode"
    per = decode_rows_per_pass(D, group_size)
    if rep_rows <= max(per, 8):
        return "decode"
    if dense:
        return "prefill"
    passes, work = -(-rep_rows // per), units * keys
    block, free, limit = (128, 3, 5 << 15) if D == 256 else (256, 4, 330_000)
    if rep_rows < block and units * passes <= 512 and (passes - free) * work <= limit:
        return "decode"
    return "prefill"


class DraftTree:
    """The tokens drafted after a sequence's last one, as a tree (speculative decoding): what a node sees in
    attention and where it sits.

    ``parents``: int32 [B, L] (or [L], one tree for the whole batch) on the GPU, the parent of each node: -1 for
    a child of the last token before the tree, else the index of an earlier node. Any other value makes
    the node absent, and its descendants with it: padding, where the trees of a batch are unequal. Node l is row
    S_b - L + l of the cache; it sees every key before the tree, its ancestors and itself, and an absent node
    nothing (its output row is 0).

    Built by one launch on the current stream; the layers of a step share it, as the mask of their attention
    calls (``attention.scaled_dot_product_attention(..., mask=tree)``, ``attention(..., tree=tree)``).

    ``depths`` [B, L] int32 are the nodes' depths (-1: absent). ``positions`` [1, B, L] int32, where ``starts`` (int32
    [B] on the GPU, or one int: the position of a depth-0 node) was given, are the nodes' positions for
    ``rope_axes``. ``refresh()`` launches again over the same buffers, after ``parents`` or ``starts`` were
    refilled in place (and into a graph)."""

    def __init__(self, parents: torch.Tensor, starts=None):
        self._starts = starts
        host, stream = _native(parents)
        buf = None if host is None else host.draft_tree(parents, starts, stream)
        if type(buf) is int:
            _lib.check(buf, "kvq_draft_tree")
        if buf is None:  # checked, served or refused here
            dev = _require_cuda(parents)
            if parents.dtype != torch.int32 or parents.dim() not in (1, 2) or parents.shape[-1] < 1:
                raise ValueError(f"parents must be int32 [B, L] or [L] with L >= 1, got {parents.dtype} {tuple(parents.shape)}")
            L = parents.shape[-1]
            if L > _lib.TREE_MAX_NODES:
                raise NotImplementedError(f"a tree has at most {_lib.TREE_MAX_NODES} nodes, got {L}")
            if parents.stride(-1) != 1 and L > 1:
                raise ValueError("the nodes of parents must be contiguous")
            B = 1 if parents.dim() == 1 else parents.shape[0]
            if torch.is_tensor(starts):
                if starts.dtype != torch.int32 or starts.device != dev or tuple(starts.shape) != (B,) or \
                        not starts.is_contiguous():
                    raise ValueError(f"starts must be an int or a contiguous int32 tensor of {B} entries on {dev}")
            elif starts is not None:
                self._starts = int(starts)
                if not -2 ** 31 <= self._starts < 2 ** 31 - L:
                    raise ValueError(f"start {starts} leaves the int32 positions")
        self.parents = parents
        self.device = parents.device
        self.shared = parents.dim() == 1  # one tree for any batch
        self.B, self.L = (1 if self.shared else parents.shape[0]), parents.shape[-1]
        self._words, self._nodes = (self.L + 31) // 32, self.B * self.L
        self._buf = buf
        if buf is None:
            self._buf = torch.empty(self._nodes * (self._words + (1 if starts is None else 2)), dtype=torch.int32,
                                    device=self.device)
            self.refresh()

    @functools.cached_property
    def bits(self) -> torch.Tensor:
        return self._buf[: self._nodes * self._words].view(self.B, self.L, self._words)

    @functools.cached_property
    def depths(self) -> torch.Tensor:
        n = self._nodes * self._words
        return self._buf[n: n + self._nodes].view(self.B, self.L)

    @functools.cached_property
    def positions(self) -> Optional[torch.Tensor]:
        n = self._nodes * (self._words + 1)
        return None if self._starts is None else self._buf[n:].view(1, self.B, self.L)

    @functools.cached_property
    def desc(self) -> "_lib.Tree":
        at = self._buf.data_ptr()
        return _lib.Tree(at, at + 4 * self._nodes * self._words, 0 if self.shared else self.L * self._words,
                         0 if self.shared else self.L)

    def refresh(self) -> None:
        tensor = torch.is_tensor(self._starts)
        with _on_device(self.device):
            rc = _lib.lib().kvq_draft_tree(
                self.parents.data_ptr(), 0 if self.shared else self.parents.stride(0), self.B, self.L, self.desc.bits,
                self.desc.depths, self._starts.data_ptr() if tensor else None,
                0 if tensor or self._starts is None else self._starts,
                None if self._starts is None else self.positions.data_ptr(), _lib.stream_ptr(self.device))
        _lib.check(rc, "kvq_draft_tree")

    def check(self, B: int, L: int, device) -> None:
        """Raise unless queries [B, *, L, *] on `device` can be this tree's nodes."""
        if self.L != L or (not self.shared and self.B != B) or self.device != device:
            raise ValueError(f"the tree has {self.L} nodes for a batch of {'any' if self.shared else self.B} on "
                             f"{self.device}; the queries are {L} rows for {B} on {device}")


class AttentionCall:
    """A validated attention launch with its C-ABI arguments built once.

    ``prepare_attention`` checks shapes and dtypes, sizes the workspace and packs the ctypes
    descriptors; calling the object launches the kernels on the stream that was current at
    preparation time, with no further host-side work beyond one foreign call. Tensors are held
    by reference, so refilling them in place (a new query, appended cache rows inside the same
    views) is picked up by the next launch. Used by serving loops and HIP-graph capture.
    """

    def __init__(self, fn, args, keep, kernel: str, out: torch.Tensor, symbol: str):
        self._fn = fn
        self._args = args
        self._keep = keep  # tensors and ctypes structs whose addresses are baked into _args
        self.kernel = kernel  # "decode" or "prefill"
        self.symbol = symbol  # the C entry point
        self.out = out

    def __call__(self) -> torch.Tensor:
        rc = self._fn(*self._args)
        if rc:
            _lib.check(rc, self.symbol)
        return self.out


def _rows_ok(t: torch.Tensor) -> bool:
    """Rows the kernels can read directly: unit stride, 16-byte aligned, strides of 8 elements."""
    return t.stride(-1) == 1 and not any(st % 8 for st in t.stride()[:3]) and t.data_ptr() % 16 == 0


def _check_out(out: Optional[torch.Tensor], queries: torch.Tensor, dev) -> torch.Tensor:
    """A fresh output, or the caller's after the checks the kernels' stores rely on: the queries'
    shape, dtype and device, unit stride along D, 8-byte alignment and strides of 4 elements (the
    kernels write 4 elements at a time; prefill also needs 16-byte rows, checked by the library)."""
    B, Hq, L, D = queries.shape
    if out is None:
        return torch.empty((B, Hq, L, D), dtype=queries.dtype, device=dev)
    if tuple(out.shape) != (B, Hq, L, D) or out.dtype != queries.dtype or out.device != dev:
        raise ValueError(f"out must be a {queries.dtype} tensor of shape {(B, Hq, L, D)} on {dev}")
    if out.stride(-1) != 1 or any(st % 4 for st in out.stride()[:3]) or out.data_ptr() % 8:
        raise ValueError("out must have unit stride along D, 8-byte alignment and strides that are multiples of 4")
    return out


def _copy_for_one_shot(t: torch.Tensor, name: str, one_shot: bool) -> torch.Tensor:
    """A contiguous copy of a tensor the kernels cannot read in place. Only a one-shot call may take
    it: a prepared call holds its tensors by reference, so a copy would silently freeze them."""
    if not one_shot:
        raise ValueError(
            f"prepare_attention: {name} need unit stride along D, 16-byte alignment and strides that are multiples "
            f"of 8 elements (got strides {tuple(t.stride())}); a prepared call reads its tensors in place on every "
            f"launch, so pass .contiguous() tensors (and refill those)")
    return t.contiguous()


def prepare_attention(queries: torch.Tensor, keys, values, scale: float, *, causal: bool = False,
                      window: int = 0, seq_lens: Optional[torch.Tensor] = None, group_size: int = 64,
                      bits: int = 8, out: Optional[torch.Tensor] = None, kernel: str = "auto",
                      workspace: Optional[torch.Tensor] = None, tree: Optional[DraftTree] = None,
                      _one_shot: bool = False) -> AttentionCall:
    """Validate one attention launch and return it as an ``AttentionCall`` (see ``attention``).

    The queries and unquantized keys/values must be readable in place (unit stride along D, 16-byte
    aligned, strides in multiples of 8 elements): a prepared call reads the same memory on every
    launch, so a tensor that would need a copy raises ValueError rather than being snapshotted."""
    if queries.dim() != 4:
        raise ValueError(f"queries must be [B, Hq, L, D], got {tuple(queries.shape)}")
    B, Hq, L, D = queries.shape
    dense = torch.is_tensor(keys)
    if dense:
        if not torch.is_tensor(values):
            raise ValueError("keys and values must both be tensors (unquantized) or both be triples")
        dev = _require_cuda(queries, keys, values)
        Hkv, S = keys.shape[1], keys.shape[2]
        for name, t in (("keys", keys), ("values", values)):
            if t.dim() != 4 or tuple(t.shape) != (B, Hkv, S, D):
                raise ValueError(f"{name} must be [B, Hkv, S, D] = {(B, Hkv, S, D)}, got {tuple(t.shape)}")
            if t.dtype != queries.dtype:
                raise ValueError(f"{name} are {t.dtype}, queries are {queries.dtype}")
        if not _rows_ok(keys):
            keys = _copy_for_one_shot(keys, "keys", _one_shot)
        if not _rows_ok(values):
            values = _copy_for_one_shot(values, "values", _one_shot)
    else:
        _check_triple(keys, "keys")
        _check_triple(values, "values")
        dev = _require_cuda(queries, *keys, *values)
        Hkv, S = keys[0].shape[1], keys[0].shape[2]
        for name, tr in (("keys", keys), ("values", values)):
            c, s, b = tr
            if c.shape[0] != B or c.shape[1] != Hkv or c.shape[2] != S or s.shape[:3] != c.shape[:3]:
                raise ValueError(f"{name} triple shapes {tuple(c.shape)}, {tuple(s.shape)} do not match B={B}, Hkv={Hkv}, S={S}")
            if c.shape[3] * 32 // bits != D:
                raise ValueError(f"{name} codes hold {c.shape[3] * 32 // bits} dims at {bits} bits, queries have {D}")
            if s.shape[3] * group_size != D:
                raise ValueError(f"{name} scales hold {s.shape[3]} groups, expected D/group_size = {D // group_size}")
            if s.dtype != queries.dtype:
                raise ValueError(f"{name} scales are {s.dtype}, queries are {queries.dtype}")
    if Hq % Hkv:
        raise ValueError(f"Hq={Hq} is not a multiple of Hkv={Hkv}")
    if not _rows_ok(queries):
        queries = _copy_for_one_shot(queries, "queries", _one_shot)
    out = _check_out(out, queries, dev)
    sl_ptr = None
    if seq_lens is not None:
        if seq_lens.dtype != torch.int32 or seq_lens.device != dev or seq_lens.numel() != B:
            raise ValueError("seq_lens must be an int32 tensor of B entries on the queries' device")
        sl_ptr = seq_lens.data_ptr()
    rep = Hq // Hkv
    if tree is not None:
        return _prepare_tree(queries, keys, values, scale, tree, out, dense=dense, window=window, seq_lens=seq_lens,
                             group_size=group_size, bits=bits, causal=causal, kernel=kernel, workspace=workspace,
                             one_shot=_one_shot)
    if kernel == "auto":
        kernel = _auto_kernel(rep * L, D, 64 if dense else group_size, dense=dense, units=B * Hkv,
                              keys=min(S, window + L) if window else S)
    if kernel not in ("decode", "prefill"):
        raise ValueError(f"kernel must be 'decode', 'prefill' or 'auto', got {kernel!r}")
    lib = _lib.lib()
    ws_fn = lib.kvq_decode_workspace_size if kernel == "decode" else lib.kvq_prefill_workspace_size
    symbol = f"kvq_{kernel}_attn" + ("_dense" if dense else "")
    fn = getattr(lib, symbol)
    nbytes = ws_fn(B, Hq, Hkv, L, D, S, int(window))
    if nbytes == 0:
        raise NotImplementedError(f"{kernel} attention does not support B={B} Hq={Hq} Hkv={Hkv} L={L} D={D} S={S}")
    stream = _lib.stream_ptr(dev)
    if workspace is None:
        ws = _workspace(dev, stream, nbytes)
    else:
        if workspace.device != dev or workspace.numel() * workspace.element_size() < nbytes:
            raise ValueError(f"workspace must hold at least {nbytes} bytes on {dev}")
        ws = workspace
    qr, orr = _lib.rows(queries), _lib.rows(out)
    tail = (_lib.dtype_code(queries.dtype), float(scale), int(bool(causal)), int(window), ws.data_ptr(),
            ws.numel() * ws.element_size(), stream)
    if dense:
        kq, vq = _lib.rows(keys), _lib.rows(values)
        args = (ctypes.byref(qr), ctypes.byref(kq), ctypes.byref(vq), sl_ptr, ctypes.byref(orr), B, Hq, Hkv, L, D, S,
                *tail)
    else:
        # the caches' range words: registered with their buffers, else (one-shot bf16 prefill calls)
        # computed from the scales and biases on the device; decode applies scales in fp32 and
        # reads none, and an fp16 cache's values always fit the operands
        kw, vw = range_word(keys[0]), range_word(values[0])
        if kernel == "prefill" and _one_shot and queries.dtype == torch.bfloat16:
            kw = range_exponent(keys, bits) if kw is None else kw
            vw = range_exponent(values, bits) if vw is None else vw
        kq, vq = _lib.qtensor(*keys, range_exp=kw), _lib.qtensor(*values, range_exp=vw)
        args = (ctypes.byref(qr), ctypes.byref(kq), ctypes.byref(vq), sl_ptr, ctypes.byref(orr), B, Hq, Hkv, L, D, S,
                int(bits), int(group_size), *tail)
        keep_words = (kw, vw)
    keep = (queries, keys, values, seq_lens, ws, qr, orr, kq, vq) + (() if dense else keep_words)
    return AttentionCall(fn, args, keep, kernel, out, symbol)


_COUNTER_BYTES = 1 << 18  # the arrival counters at the start of a workspace, zero before its first call


def _tree_workspace(dev: torch.device, stream: int, nbytes: int, workspace: Optional[torch.Tensor]) -> torch.Tensor:
    """The caller's workspace after its checks, or the stream's. A call that is captured into a graph without one
    gets its own from the graph's memory (its counters cleared by a fill in every replay): graphs that were
    captured on one stream may be replayed at once on others."""
    if workspace is not None:
        if workspace.device != dev or not workspace.is_contiguous() or \
                workspace.numel() * workspace.element_size() < nbytes:
            raise ValueError(f"workspace must hold at least {nbytes} contiguous bytes on {dev}")
        return workspace
    if torch.cuda.is_current_stream_capturing():
        ws = torch.empty(max(nbytes, _COUNTER_BYTES), dtype=torch.uint8, device=dev)
        ws[:_COUNTER_BYTES].zero_()
        return ws
    return _workspace(dev, stream, nbytes)


class _DeviceCall(AttentionCall):
    """An AttentionCall whose launch makes its tensors' device the current one."""

    def __init__(self, dev: torch.device, *args):
        super().__init__(*args)
        self._dev = dev

    def __call__(self) -> torch.Tensor:
        with _on_device(self._dev):
            return super().__call__()


def _check_tree_call(tree: DraftTree, B: int, L: int, S: int, window: int, causal: bool, kernel: str, device) -> None:
    tree.check(B, L, device)
    if causal or kernel != "auto":
        raise ValueError("a tree says what its nodes see and which kernel serves them: no causal= or kernel= with tree=")
    if S < L:
        raise ValueError(f"the tree's {L} nodes are the last rows of the cache, which has {S}")
    if window < 0:
        raise ValueError(f"window must be >= 0, got {window}")


@functools.lru_cache(maxsize=256)
def _tree_sizes(*sizes: int) -> Tuple[int, bool]:
    """(workspace bytes, whether a bf16 cache's range words are read) of a tree call, which follow from its sizes."""
    B, Hq, Hkv, L, D, S, bits, group_size, window = sizes
    lib = _lib.lib()
    return (lib.kvq_tree_workspace_size(B, Hq, Hkv, L, D, S, window),
            lib.kvq_tree_kernel(B, Hq, Hkv, L, D, S, bits, group_size, window) == _lib.TREE_PREFILL)


def _prepare_tree(queries, keys, values, scale, tree, out, *, dense, window, seq_lens, group_size, bits, causal, kernel,
                  workspace, one_shot) -> AttentionCall:
    """prepare_attention's call over a tree (its tensors have been checked there)."""
    B, Hq, L, D = queries.shape
    dev = queries.device
    Hkv, S = keys.shape[1:3] if dense else keys[0].shape[1:3]
    _check_tree_call(tree, B, L, S, window, causal, kernel, dev)
    nbytes, ranges = _tree_sizes(B, Hq, Hkv, L, D, S, 16 if dense else int(bits), 64 if dense else int(group_size), int(window))
    if nbytes == 0:
        raise NotImplementedError(f"tree attention does not support B={B} Hq={Hq} Hkv={Hkv} L={L} D={D} S={S}")
    stream = _lib.stream_ptr(dev)
    with _on_device(dev):
        ws = _tree_workspace(dev, stream, nbytes, workspace)
    qr, orr = _lib.rows(queries), _lib.rows(out)
    kw = vw = None
    if dense:
        symbol, kq, vq, form = "kvq_tree_attn_dense", _lib.rows(keys), _lib.rows(values), ()
    else:
        # a bf16 cache's range words, as prepare_attention has them
        if ranges and queries.dtype == torch.bfloat16:
            kw, vw = range_word(keys[0]), range_word(values[0])
            if one_shot:
                kw = range_exponent(keys, bits) if kw is None else kw
                vw = range_exponent(values, bits) if vw is None else vw
        symbol, form = "kvq_tree_attn", (int(bits), int(group_size))
        kq, vq = _lib.qtensor(*keys, range_exp=kw), _lib.qtensor(*values, range_exp=vw)
    args = (ctypes.byref(qr), ctypes.byref(kq), ctypes.byref(vq), None if seq_lens is None else seq_lens.data_ptr(),
            ctypes.byref(orr), B, Hq, Hkv, L, D, S, *form, _lib.dtype_code(queries.dtype), float(scale),
            ctypes.byref(tree.desc), int(window), ws.data_ptr(), ws.numel() * ws.element_size(), stream)
    keep = (queries, keys, values, seq_lens, ws, qr, orr, kq, vq, tree, kw, vw)
    return _DeviceCall(dev, getattr(_lib.lib(), symbol), args, keep, "tree", out, symbol)


def _tree_attention(queries, keys, values, scale, tree: DraftTree, window, seq_lens, group_size, bits, table=None,
                    max_len=None) -> Optional[torch.Tensor]:
    """Attention over a tree through the native host path (`keys` and `values` are pools with a block table); None for a
    call it does not take, and under capture, where the call has a workspace of its own."""
    host, stream = _native(queries)
    if host is None or type(window) is not int or torch.cuda.is_current_stream_capturing():
        return None
    dev = queries.get_device()
    head = (queries, keys, values, scale, window, seq_lens, group_size, bits, _range_words)
    tail = (stream, tree._buf, 0 if tree.shared else tree.B, tree.L, table, -1 if max_len is None else max_len)
    out = host.tree_attention(*head, _workspaces.get((dev, stream)), *tail)
    if type(out) is int and out > 0:  # the bytes of workspace it needs
        out = host.tree_attention(*head, _workspace(queries.device, stream, out), *tail)
    if type(out) is int:  # a failed launch, which is not tried again
        _lib.check(out, "kvq_tree_attn" if table is None else "kvq_paged_tree_attn")
    return out


def layer_attention(queries: torch.Tensor, keys, values, scale: float, *, causal: bool, window: int = 0,
                    seq_lens: Optional[torch.Tensor] = None, group_size: int = 64,
                    bits: int = 8) -> Optional[torch.Tensor]:
    """``attention`` over a quantized cache through the native host path, for the calls a model's layers
    make (the same checks, kernels and results); None for any other form, which ``attention`` then serves
    or refuses."""
    if not (torch.is_tensor(queries) and queries.is_cuda and queries.dim() == 4 and type(keys) is tuple and
            type(values) is tuple and len(keys) == 3):
        return None
    B, Hq, L, D = queries.shape
    if D not in NATIVE_HEAD_DIMS and D != 96:
        return None
    Hkv, S = keys[0].shape[1:3] if keys[0].dim() == 4 else (0, 0)
    if not Hkv or Hq % Hkv or group_size not in (32, 64, 128) or type(window) is not int:
        return None
    prefill = _auto_kernel(Hq // Hkv * L, D, group_size, dense=False, units=B * Hkv,
                           keys=min(S, window + L) if window else S) == "prefill"
    kw = vw = None
    if prefill and queries.dtype == torch.bfloat16:  # the range words, which only these kernels read
        kw, vw = range_word(keys[0]), range_word(values[0])
        if kw is None or vw is None:
            return None
    dev = queries.device.index
    stream = torch._C._cuda_getCurrentRawStream(dev)
    ws = _workspaces.get((dev, stream))
    args = (queries, keys, values, float(scale), int(causal), window, seq_lens, group_size, bits, int(prefill),
            0 if kw is None else kw.data_ptr(), 0 if vw is None else vw.data_ptr())
    call = _lib.host().attention
    out = call(*args, ws, stream)
    if type(out) is int and out > 0:  # the bytes of workspace it needs
        out = call(*args, _workspace(queries.device, stream, out), stream)
    if type(out) is int:  # a failed launch, which is not tried again
        _lib.check(out, "kvq_prefill_attn" if prefill else "kvq_decode_attn")
    return out


def attention(queries: torch.Tensor, keys, values, scale: float, *, causal: bool = False,
              window: int = 0, seq_lens: Optional[torch.Tensor] = None, group_size: int = 64, bits: int = 8,
              out: Optional[torch.Tensor] = None, kernel: str = "auto",
              tree: Optional[DraftTree] = None) -> torch.Tensor:
    """softmax(scale * q K^T + mask) V. queries [B, Hq, L, D]; keys/values either quantized triples
    (codes [B, Hkv, S, D*bits/32], scales/biases [B, Hkv, S, D/G]) or unquantized tensors
    [B, Hkv, S, D] in the queries' dtype; returns [B, Hq, L, D] (or fills `out`). kernel: "decode",
    "prefill" or "auto" (decode while a KV head's query rows fit max(16*G/D, 8) columns, and past
    that where its passes over the keys cost less than the prefill kernel's row blocks).

    With `tree` the queries are the nodes of a DraftTree, whose keys are each sequence's last L rows (of
    seq_lens[b] >= L, or of S); a window must then be at least L, and the scale positive."""
    if tree is not None and out is None and kernel == "auto" and not causal:
        got = _tree_attention(queries, keys, values, scale, tree, window, seq_lens, group_size, bits)
        if got is not None:
            return got
    return prepare_attention(queries, keys, values, scale, causal=causal, window=window, seq_lens=seq_lens,
                             group_size=group_size, bits=bits, out=out, kernel=kernel, tree=tree, _one_shot=True)()


# ---- general masks (kvq_mask): boolean masks with no causal / window / padding structure, per-head
# masks and additive masks, read by the decode kernel beside every tile

_MASK_KINDS = {torch.bool: _lib.MASK_BOOL, torch.float16: _lib.MASK_F16, torch.bfloat16: _lib.MASK_BF16,
               torch.float32: _lib.MASK_F32}


def mask_view(mask: torch.Tensor, B: int, Hq: int, Hkv: int, L: int, S: int, layout: str = "heads"):
    """The mask as the kernels read it: (tensor, (stride_b, stride_kvh, stride_rep, stride_l)) over the
    [B, Hkv, Hq / Hkv, L, S] score layout, keys contiguous, broadcast dimensions at stride 0.

    ``layout`` is how the caller's reference broadcasts the mask against the scores:
      "heads"    against [B, Hq, L, S] (mx.fast.scaled_dot_product_attention);
      "grouped"  against [B, Hkv, Hq / Hkv, L, S] as given (mlx-lm's quantized SDPA, the L == 1 /
                 short-S hand-off of m5engine/attention.py:42-45);
      "blocked"  a mask of rank 3 or more gains an axis at -3 first (m5engine/attention.py:55-56),
                 so its head axis indexes KV heads.
    With Hq == Hkv the three agree."""
    if layout not in ("heads", "grouped", "blocked"):
        raise ValueError(f"layout must be 'heads', 'grouped' or 'blocked', got {layout!r}")
    m = mask
    if m.dtype == torch.float64:
        m = m.float()
    if m.dtype not in _MASK_KINDS:
        raise ValueError(f"masks are bool (visible keys) or float (additive), got {m.dtype}")
    if m.dim() == 0 or m.shape[-1] not in (1, S):
        raise ValueError(f"the mask's last dimension {tuple(m.shape)[-1:]} does not broadcast to S = {S}")
    if m.shape[-1] == 1 and S != 1:
        m = m.expand(*m.shape[:-1], S)
    if m.stride(-1) != 1:
        m = m.contiguous()
    rep = Hq // Hkv
    try:
        if rep == 1 or layout == "heads":
            m4 = torch.broadcast_to(m, (B, Hq, L, S))
            sb, sh, sl, _ = m4.stride()
            return m4, (sb, rep * sh, sh, sl)
        if layout == "blocked" and m.dim() >= 3:
            m = m.unsqueeze(-3)
        m5 = torch.broadcast_to(m, (B, Hkv, rep, L, S))
    except RuntimeError as e:
        raise ValueError(f"mask of shape {tuple(mask.shape)} does not broadcast to the scores: {e}") from None
    sb, skv, srep, sl, _ = m5.stride()
    return m5, (sb, skv, srep, sl)


@functools.lru_cache(maxsize=256)
def _masked_on_prefill(*sizes: int) -> int:
    """kvq_masked_on_prefill, which follows from the sizes alone (a layer's foreign call costs 0.5 us)."""
    return _lib.lib().kvq_masked_on_prefill(*sizes)


def masked_attention(queries: torch.Tensor, keys, values, scale: float, mask: torch.Tensor, *, layout: str = "heads",
                     group_size: int = 64, bits: int = 8, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale * q K^T + mask) V under a general mask (boolean: visible keys; float: added to
    the scores), keys/values quantized triples or unquantized tensors as for ``attention``. Runs the
    decode kernel (rows beyond one pass take more passes over the keys), the prefill kernel where it
    has the mask's form (boolean, and additive over unquantized caches) and the rows and keys are
    many, or, for an unquantized head_dim-256 cache, the head_dim-256 kernel. A row that sees no key returns 0."""
    if queries.dim() != 4:
        raise ValueError(f"queries must be [B, Hq, L, D], got {tuple(queries.shape)}")
    B, Hq, L, D = queries.shape
    dense = torch.is_tensor(keys)
    if dense:
        dev = _require_cuda(queries, keys, values)
        Hkv, S = keys.shape[1], keys.shape[2]
        for name, t in (("keys", keys), ("values", values)):
            if t.dim() != 4 or tuple(t.shape) != (B, Hkv, S, D) or t.dtype != queries.dtype:
                raise ValueError(f"{name} must be {queries.dtype} [B, Hkv, S, D] = {(B, Hkv, S, D)}")
        keys = keys if _rows_ok(keys) else keys.contiguous()
        values = values if _rows_ok(values) else values.contiguous()
    else:
        _check_triple(keys, "keys")
        _check_triple(values, "values")
        dev = _require_cuda(queries, *keys, *values)
        Hkv, S = keys[0].shape[1], keys[0].shape[2]
        if keys[0].shape[0] != B or keys[0].shape[3] * 32 // bits != D or keys[1].shape[3] * group_size != D:
            raise ValueError("keys triple does not match the queries' B and D at these bits and group_size")
    if Hq % Hkv:
        raise ValueError(f"Hq={Hq} is not a multiple of Hkv={Hkv}")
    if not torch.is_tensor(mask):
        raise ValueError("mask must be a tensor")
    if mask.device != dev:
        mask = mask.to(dev)
    mview, strides = mask_view(mask, B, Hq, Hkv, L, S, layout)
    desc = _lib.Mask(mview.data_ptr(), _MASK_KINDS[mview.dtype], *strides)
    if not _rows_ok(queries):
        queries = queries.contiguous()
    out = _check_out(out, queries, dev)
    lib = _lib.lib()
    stream = _lib.stream_ptr(dev)
    qr, orr = _lib.rows(queries), _lib.rows(out)
    if dense:
        symbol, fn = "kvq_decode_attn_dense_masked", lib.kvq_decode_attn_dense_masked
        kr, vr = _lib.rows(keys), _lib.rows(values)
        sizes = (B, Hq, Hkv, L, D, S, _lib.dtype_code(queries.dtype))
    else:
        symbol, fn = "kvq_decode_attn_masked", lib.kvq_decode_attn_masked
        kw = vw = None
        # a bf16 cache's range words, which only the prefill kernel reads
        if queries.dtype == torch.bfloat16 and _masked_on_prefill(B, Hq, Hkv, L, D, S):
            kw, vw = range_word(keys[0]), range_word(values[0])
        kr, vr = _lib.qtensor(*keys, range_exp=kw), _lib.qtensor(*values, range_exp=vw)
        sizes = (B, Hq, Hkv, L, D, S, int(bits), int(group_size), _lib.dtype_code(queries.dtype))
    args = (ctypes.byref(qr), ctypes.byref(kr), ctypes.byref(vr), ctypes.byref(orr), *sizes, float(scale), ctypes.byref(desc))
    # the stream's workspace as it is: the library plans the call anyway and says if it is too small (asking
    # first costs 1 us of the 8 to 10 us that a short call takes on the device)
    ws = _workspaces.get((dev.index, stream))
    rc = _lib.ERR_WORKSPACE if ws is None else fn(*args, ws.data_ptr(), ws.numel(), stream)
    if rc in (_lib.ERR_WORKSPACE, _lib.ERR_INVALID):
        nbytes = lib.kvq_decode_workspace_size(B, Hq, Hkv, L, D, S, 0)
        if nbytes == 0:
            raise NotImplementedError(f"decode attention does not support B={B} Hq={Hq} Hkv={Hkv} L={L} D={D} S={S}")
        if rc == _lib.ERR_WORKSPACE:
            ws = _workspace(dev, stream, nbytes)
            rc = fn(*args, ws.data_ptr(), ws.numel(), stream)
    if rc:
        _lib.check(rc, symbol)
    return out


# ---- paged pools (64-row pages; include/kvq.h "Paged layout")

PAGE_ROWS = _lib.PAGE_ROWS


def _check_table(block_tables: torch.Tensor, B: int, dev) -> None:
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] != B:
        raise ValueError(f"block_tables must be int32 [B={B}, max_pages], got {block_tables.dtype} "
                         f"{tuple(block_tables.shape)}")
    if block_tables.device != dev or block_tables.stride(1) != 1:
        raise ValueError("block_tables must be on the queries' device with contiguous rows")


def _whole_table(block_tables: torch.Tensor, B: int, dev) -> torch.Tensor:
    """A checked table whose rows follow each other: the library takes the distance of its rows for their length, so
    a view of a wider table's first pages is copied, lest the entries behind it be taken for the sequence's."""
    _check_table(block_tables, B, dev)
    return block_tables if block_tables.stride(0) == block_tables.shape[1] else block_tables.contiguous()


def paged_quantize_append(k: torch.Tensor, k_pool: Triple, v: Optional[torch.Tensor], v_pool: Optional[Triple],
                          block_tables: torch.Tensor, *, starts: Optional[torch.Tensor] = None, row_offset: int = 0,
                          group_size: int = 64, bits: int = 8, rope: Optional[Rope] = None) -> None:
    """Quantize k (and v) [B, H, L, D] into paged pools ([num_pages, H, 64, *] triples): row l of
    sequence b goes to row starts[b] + l (or row_offset + l) of that sequence's pages. With `rope`
    the keys are rotated at those positions first."""
    _check_triple(k_pool, "k_pool")
    tens = [k, *k_pool]
    if v is not None:
        _check_triple(v_pool, "v_pool")
        tens += [v, *v_pool]
    dev = _require_cuda(*tens)
    B, H, L, D = k.shape
    _check_table(block_tables, B, dev)
    st_ptr = None
    if starts is not None:
        if starts.dtype != torch.int32 or starts.numel() != B or starts.device != dev:
            raise ValueError("starts must be an int32 tensor of B entries on the same device")
        st_ptr = starts.data_ptr()
    kr, kq = _lib.rows(k), _lib.qtensor(*k_pool, range_exp=range_word(k_pool[0]))
    vr_p = vq_p = None
    if v is not None:
        vr, vq = _lib.rows(v), _lib.qtensor(*v_pool, range_exp=range_word(v_pool[0]))
        vr_p, vq_p = ctypes.byref(vr), ctypes.byref(vq)
    rp = None
    if rope is not None:
        rparams = rope.params(0 if starts is not None else row_offset)
        rp = ctypes.byref(rparams)
    rc = _lib.lib().kvq_paged_quantize_append(
        ctypes.byref(kr), ctypes.byref(kq), vr_p, vq_p, k_pool[0].shape[0], block_tables.data_ptr(),
        block_tables.stride(0), st_ptr, int(row_offset), rp, B, H, L, D, int(bits), int(group_size),
        _lib.dtype_code(k.dtype), _lib.stream_ptr(dev))
    _lib.check(rc, "kvq_paged_quantize_append")


def _check_starts(starts: Optional[torch.Tensor], B: int, dev) -> Optional[int]:
    if starts is None:
        return None
    if starts.dtype != torch.int32 or tuple(starts.shape) != (B,) or starts.device != dev or not starts.is_contiguous():
        raise ValueError("starts must be a contiguous int32 tensor of B entries on the same device")
    return starts.data_ptr()


def paged_rope_axes_append(k: torch.Tensor, k_pool: Triple, v: Optional[torch.Tensor], v_pool: Optional[Triple],
                           block_tables: torch.Tensor, rope: RopeAxes, positions: torch.Tensor, *,
                           starts: Optional[torch.Tensor] = None, row_offset: int = 0,
                           queries: Optional[torch.Tensor] = None, group_size: int = 64, bits: int = 8) -> None:
    """``paged_quantize_append`` with the keys rotated at `positions` (int32 [axes, B, L]) first, and the rows of
    `queries` [B, Hq, L, D] rotated in place in the same launch."""
    AxesAppendCall(k_pool, v_pool, rope, group_size, bits).paged(k, v, positions, block_tables, starts, row_offset, queries)


def paged_dequantize(k_pool: Triple, v_pool: Optional[Triple], block_tables: torch.Tensor, seq_lens: torch.Tensor, *,
                     group_size: int = 64, bits: int = 8, max_len: Optional[int] = None, out=None):
    """The first seq_lens[b] rows of every sequence, read back through its block table: (K, V) [B, H, max_len, D]
    (or (K,) without v_pool). max_len bounds seq_lens (default: out's rows, else the table's capacity). Rows behind
    a sequence are left as they are in `out`, and are 0 in new tensors."""
    if out is not None and v_pool is not None and type(k_pool) is tuple and len(out) == 2:
        out = tuple(out)
        got = read_rows(k_pool, v_pool, 0, out[0].shape[2] if max_len is None else int(max_len), group_size=group_size,
                        bits=bits, out=out, table=block_tables, seq_lens=seq_lens)
        if got is not None:
            return got
    dev, (_, H, rows), D = _check_read(k_pool, v_pool, group_size, bits)
    if rows != PAGE_ROWS:
        raise ValueError(f"pools must be [num_pages, H, {PAGE_ROWS}, *]")
    B = block_tables.shape[0]
    block_tables = _whole_table(block_tables, B, dev)
    if seq_lens.dtype != torch.int32 or tuple(seq_lens.shape) != (B,) or seq_lens.device != dev or not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be a contiguous int32 tensor of B entries on the pools' device")
    if max_len is None:
        max_len = block_tables.shape[1] * PAGE_ROWS if out is None else tuple(out)[0].shape[2]
    n = int(max_len)
    outs = _read_out(out, 1 if v_pool is None else 2, (B, H, n, D), k_pool[1].dtype, dev, torch.zeros)
    if outs[0].numel() == 0:
        return outs
    kq, kr = _lib.qtensor(*k_pool), _lib.rows(outs[0])
    vq, vr = (None, None) if v_pool is None else (_lib.qtensor(*v_pool), _lib.rows(outs[1]))
    ref = ctypes.byref
    with _on_device(dev):
        rc = _lib.lib().kvq_paged_dequantize(
            ref(kq), ref(kr), None if vq is None else ref(vq), None if vr is None else ref(vr), k_pool[0].shape[0],
            block_tables.data_ptr(), block_tables.stride(0), seq_lens.data_ptr(), B, H, n, D, int(bits), int(group_size),
            _lib.dtype_code(k_pool[1].dtype), _lib.stream_ptr(dev))
    _lib.check(rc, "kvq_paged_dequantize")
    return outs


# ---- keeping accepted rows

def _row_arrays(tensors) -> "ctypes.Array":
    arr = (_lib.RowArray * len(tensors))()
    for a, t in zip(arr, tensors):
        n = t.element_size()
        a.data, a.row_bytes = t.data_ptr(), t.shape[3] * n
        a.stride_b, a.stride_h, a.stride_l = (n * s for s in t.stride()[:3])
    return arr


def _check_kept(tensors, rows: torch.Tensor, B: int, n: Optional[int]):
    if not tensors:
        raise ValueError("no cache arrays")
    dev = _require_cuda(*tensors, rows)
    H = tensors[0].shape[1]
    for t in tensors:
        if t.dim() != 4 or t.shape[1] != H or t.stride(3) != 1:
            raise ValueError(f"cache arrays must be 4-D [*, {H}, rows, width] with contiguous rows, got {tuple(t.shape)}")
    if rows.dtype != torch.int32 or rows.dim() not in (1, 2) or (rows.dim() == 2 and rows.shape[0] != B) or \
            (rows.shape[-1] > 1 and rows.stride(-1) != 1):
        raise ValueError(f"rows must be int32 [B={B}, M] or [M] with contiguous entries, got {rows.dtype} {tuple(rows.shape)}")
    M = rows.shape[-1]
    return dev, H, M, (rows.stride(0) if rows.dim() == 2 else 0)


def move_rows(tensors, rows, start: int, n: int, table=None, starts=None) -> bool:
    """``keep_rows``, or with a block table ``paged_keep_rows``, through the native host path, of tensors in nested lists and
    tuples; False for a call it does not take."""
    host, stream = _native(rows)
    done = None if host is None else host.keep_rows(tensors, rows, start, n, table, starts, stream)
    if done is not None and done is not True:
        _lib.check(done, "kvq_keep_rows")
    return done is True


def keep_rows(tensors: Sequence[torch.Tensor], rows: torch.Tensor, start: int, n: int) -> None:
    """Move the accepted rows of drafted ones up, in place: in every array [B, H, cap, W] of `tensors` (codes, scales,
    biases, or unquantized rows; any mix of layers), row start + i of sequence b becomes what row start + rows[b, i] held,
    for the M entries of rows (int32 [B, M] or [M], on the GPU; indices among the n rows from `start`). An entry outside
    [i, n) leaves its row as it is, so an ascending list padded with -1 keeps fewer rows for some sequences. An array named
    twice, or broadcast, is refused. One launch for up to 192 arrays."""
    tensors = list(tensors)
    if move_rows(tensors, rows, start, n):
        return
    B = tensors[0].shape[0] if tensors else 0
    dev, H, M, sb = _check_kept(tensors, rows, B, n)
    if any(t.shape[0] != B or start < 0 or start + n > t.shape[2] for t in tensors):
        raise ValueError(f"every array must hold {B} sequences and rows [{start}, {start + n})")
    if M == 0:
        return
    arr = _row_arrays(tensors)
    with _on_device(dev):
        rc = _lib.lib().kvq_keep_rows(arr, len(tensors), 0, None, 0, rows.data_ptr(), sb, None, int(start), int(n), M, B, H,
                                      _lib.stream_ptr(dev))
    _lib.check(rc, "kvq_keep_rows")


def paged_keep_rows(pools: Sequence[Tuple[Triple, Triple]], block_tables: torch.Tensor, rows: torch.Tensor, *,
                    starts: Optional[torch.Tensor] = None, start: int = 0, n: Optional[int] = None) -> None:
    """``keep_rows`` over paged pools: `pools` are the layers' (K triple, V triple); sequence b's drafted rows begin at
    row starts[b] (int32 [B] on the GPU; default: `start` for all). `n`: how many were drafted (default: any row of the
    table may be named). A row outside the table, or on a page outside the pool, is neither read nor written."""
    if n is None and torch.is_tensor(block_tables) and block_tables.dim() == 2 and torch.is_tensor(rows) and rows.dim():
        n = max(rows.shape[-1], block_tables.shape[1] * PAGE_ROWS)
    if n is not None and move_rows(pools, rows, start, n, block_tables, starts):
        return
    tensors = [t for layer in pools for tr in layer for t in tr]
    B = block_tables.shape[0]
    dev, H, M, sb = _check_kept(tensors, rows, B, n)
    block_tables = _whole_table(block_tables, B, dev)
    pages = tensors[0].shape[0]
    if any(t.shape[0] != pages or t.shape[2] != PAGE_ROWS for t in tensors):
        raise ValueError(f"pools must be [{pages}, H, {PAGE_ROWS}, *]")
    n = max(M, block_tables.shape[1] * PAGE_ROWS) if n is None else int(n)
    if M == 0:
        return
    arr = _row_arrays(tensors)
    with _on_device(dev):
        rc = _lib.lib().kvq_keep_rows(arr, len(tensors), pages, block_tables.data_ptr(), block_tables.stride(0), rows.data_ptr(),
                                      sb, _check_starts(starts, B, dev), int(start), n, M, B, H, _lib.stream_ptr(dev))
    _lib.check(rc, "kvq_keep_rows")


def paged_attention(queries: torch.Tensor, k_pool: Triple, v_pool: Triple, block_tables: torch.Tensor,
                    seq_lens: torch.Tensor, scale: float, *, causal: bool = False, window: int = 0,
                    group_size: int = 64, bits: int = 8, max_len: Optional[int] = None,
                    out: Optional[torch.Tensor] = None, kernel: str = "auto", tree: Optional[DraftTree] = None,
                    workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale * q K^T + mask) V over paged pools: sequence b holds seq_lens[b] rows in the
    pages block_tables[b]; queries [B, Hq, L, D] sit at its last L positions (or are the nodes of `tree`,
    which those rows hold; `workspace` is then the caller's, if given). max_len bounds seq_lens (default: the
    table's capacity) and sizes the split plan."""
    if tree is not None and out is None and kernel == "auto" and not causal and workspace is None:
        got = _tree_attention(queries, k_pool, v_pool, scale, tree, window, seq_lens, group_size, bits, block_tables, max_len)
        if got is not None:
            return got
    _check_triple(k_pool, "k_pool")
    _check_triple(v_pool, "v_pool")
    dev = _require_cuda(queries, *k_pool, *v_pool)
    if queries.dim() != 4:
        raise ValueError(f"queries must be [B, Hq, L, D], got {tuple(queries.shape)}")
    B, Hq, L, D = queries.shape
    _check_table(block_tables, B, dev)
    if seq_lens.dtype != torch.int32 or seq_lens.numel() != B or seq_lens.device != dev:
        raise ValueError("seq_lens must be an int32 tensor of B entries on the queries' device")
    Hkv = k_pool[0].shape[1]
    if k_pool[0].shape[2] != PAGE_ROWS or k_pool[1].dtype != queries.dtype:
        raise ValueError(f"pools must be [num_pages, Hkv, {PAGE_ROWS}, *] with scales in the queries' dtype")
    for a, b_ in zip(k_pool, v_pool):
        if tuple(a.shape) != tuple(b_.shape) or a.dtype != b_.dtype:
            raise ValueError("v_pool must match k_pool in every shape and dtype (the kernels read both through "
                             "one block table over k_pool's page count)")
    if k_pool[0].shape[3] * 32 // bits != D or k_pool[1].shape[3] * group_size != D or k_pool[1].shape[:3] != \
            k_pool[0].shape[:3]:
        raise ValueError(f"pools' row widths do not match D={D}, bits={bits} and group_size={group_size}")
    if Hq % Hkv:
        raise ValueError(f"Hq={Hq} is not a multiple of Hkv={Hkv}")
    S = int(max_len) if max_len is not None else block_tables.shape[1] * PAGE_ROWS
    if not _rows_ok(queries):
        queries = _copy_for_one_shot(queries, "queries", True)
    out = _check_out(out, queries, dev)
    if tree is not None:
        block_tables = _whole_table(block_tables, B, dev)
        _check_tree_call(tree, B, L, S, window, causal, kernel, dev)
        nbytes, _ = _tree_sizes(B, Hq, Hkv, L, D, S, int(bits), int(group_size), int(window))
        if nbytes == 0:
            raise NotImplementedError(f"tree attention does not support B={B} Hq={Hq} Hkv={Hkv} L={L} D={D} S={S}")
        stream = _lib.stream_ptr(dev)
        qr, orr = _lib.rows(queries), _lib.rows(out)
        kq = _lib.qtensor(*k_pool, range_exp=range_word(k_pool[0]))
        vq = _lib.qtensor(*v_pool, range_exp=range_word(v_pool[0]))
        with _on_device(dev):
            ws = _tree_workspace(dev, stream, nbytes, workspace)
            rc = _lib.lib().kvq_paged_tree_attn(
                ctypes.byref(qr), ctypes.byref(kq), ctypes.byref(vq), k_pool[0].shape[0], block_tables.data_ptr(),
                block_tables.stride(0), seq_lens.data_ptr(), ctypes.byref(orr), B, Hq, Hkv, L, D, S, int(bits),
                int(group_size), _lib.dtype_code(queries.dtype), float(scale), ctypes.byref(tree.desc), int(window),
                ws.data_ptr(), ws.numel() * ws.element_size(), stream)
        _lib.check(rc, "kvq_paged_tree_attn")
        return out
    if workspace is not None:
        raise ValueError("a workspace of the caller's is taken with tree= only")
    if kernel == "auto":
        kernel = _auto_kernel((Hq // Hkv) * L, D, group_size, dense=False, units=B * Hkv,
                              keys=min(S, window + L) if window else S)
    lib = _lib.lib()
    ws_fn = lib.kvq_decode_workspace_size if kernel == "decode" else lib.kvq_prefill_workspace_size
    nbytes = ws_fn(B, Hq, Hkv, L, D, S, int(window))
    if nbytes == 0:
        raise NotImplementedError(f"{kernel} attention does not support B={B} Hq={Hq} Hkv={Hkv} L={L} D={D} S={S}")
    stream = _lib.stream_ptr(dev)
    ws = _workspace(dev, stream, nbytes)
    qr, orr = _lib.rows(queries), _lib.rows(out)
    # (only registered words: the unused rows of a pool's pages hold whatever was there)
    kw, vw = range_word(k_pool[0]), range_word(v_pool[0])
    kq, vq = _lib.qtensor(*k_pool, range_exp=kw), _lib.qtensor(*v_pool, range_exp=vw)
    fn = lib.kvq_paged_decode_attn if kernel == "decode" else lib.kvq_paged_prefill_attn
    rc = fn(ctypes.byref(qr), ctypes.byref(kq), ctypes.byref(vq), k_pool[0].shape[0], block_tables.data_ptr(),
            block_tables.stride(0), seq_lens.data_ptr(), ctypes.byref(orr), B, Hq, Hkv, L, D, S, int(bits),
            int(group_size), _lib.dtype_code(queries.dtype), float(scale), int(bool(causal)), int(window),
            ws.data_ptr(), ws.numel() * ws.element_size(), stream)
    _lib.check(rc, f"kvq_paged_{kernel}_attn")
    return out
