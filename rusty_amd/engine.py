"""Host-side mirror of Rusty's backend op surface over the gfx950 C ABI.

Names and argument meaning follow the reference so code written against
``rusty_backend`` reads the same here:

==============================  ==================================================
reference (rusty-backend)        here
==============================  ==================================================
``WgpuContext::new``  lib.rs:20  :class:`WgpuContext` (device, own HIP stream)
``UnifiedTensor``  lib.rs:79     :class:`UnifiedTensor` (device buffer + shape)
``ComputeEngine::new`` lib.rs:343 :class:`ComputeEngine`
``dequantize``  lib.rs:4872      :meth:`ComputeEngine.dequantize`
``affine_dequantize`` lib.rs:4939 :meth:`ComputeEngine.affine_dequantize`
``matmul``  lib.rs:4403          :meth:`ComputeEngine.matmul`
``matmul_bt``  lib.rs:4299       :meth:`ComputeEngine.matmul_bt`
``matmul_at``  lib.rs:4351       :meth:`ComputeEngine.matmul_at`
``rope`` (kernels.wgsl:60)       :meth:`ComputeEngine.rope`
(none: weights are f32)          :class:`QuantizedTensor`, :meth:`ComputeEngine.qmatmul`
==============================  ==================================================

As in the reference, ops are enqueued asynchronously on the context's stream
and ``to_vec`` waits for them.  Unlike the reference, a wrong shape raises
:class:`rusty_amd._lib.RqError` instead of reading clamped memory.
"""
from __future__ import annotations

import ctypes
import enum
import math
from dataclasses import dataclass
from typing import Sequence

import numpy as np

from . import _lib
from ._lib import call, rq_qweight


class DType(enum.Enum):
    """Element type of a device buffer.  FP32/FP16 are the reference's
    ``DType`` (lib.rs:57-76); the byte types carry quantized codes and packed
    words, which the reference passes as raw ``wgpu::Buffer``s."""

    FP32 = np.float32
    FP16 = np.float16
    I8 = np.int8
    U8 = np.uint8
    U32 = np.uint32
    I32 = np.int32
    U64 = np.uint64
    FP64 = np.float64

    def __init__(self, value):
        self.itemsize = np.dtype(value).itemsize

    __hash__ = object.__hash__  # members are singletons; Enum's own hashes the name, in Python, at every look-up

    @property
    def np(self):
        return np.dtype(self.value)


# Array types that UnifiedTensor.new keeps; numbers of any other become FP32.
# I32, U64 and FP64 buffers (offsets, lengths, masks, frequencies) are asked for by name.
_INFERRED = {d.value: d for d in (DType.FP32, DType.FP16, DType.I8, DType.U8, DType.U32)}


def _prod(shape: Sequence[int]) -> int:
    n = 1
    for s in shape:
        n *= int(s)
    return n


class WgpuContext:
    """Device context (replaces ``WgpuContext::new``, lib.rs:20-47).

    Kept under the reference's name so callers port unchanged; it owns a HIP
    context on a gfx950 device, not a wgpu adapter."""

    def __init__(self, device: int = 0):
        lib = _lib.lib()
        h = ctypes.c_void_p()
        call("rq_ctx_create", device, ctypes.byref(h))
        self._h = h
        self._lib = lib
        self.device = device
        s = ctypes.c_void_p()
        call("rq_ctx_stream", h, ctypes.byref(s))
        self.stream = s
        n = ctypes.c_int()
        call("rq_ctx_num_cus", h, ctypes.byref(n))
        self.num_cus = n.value

    @property
    def handle(self) -> ctypes.c_void_p:
        return self._h

    def sync(self) -> None:
        call("rq_sync", self._h, None)

    def close(self) -> None:
        if self._h:
            call("rq_ctx_destroy", self._h)
            self._h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()


Context = WgpuContext


class UnifiedTensor:
    """A device buffer with a host-side shape (replaces ``UnifiedTensor``,
    lib.rs:79-241).  Memory is freed when the object is collected."""

    def __init__(self, ctx: WgpuContext, ptr: int, shape: Sequence[int], dtype: DType, owner: bool = True):
        self.ctx = ctx
        self.ptr = ptr
        self.shape = tuple(int(s) for s in shape)
        self.dtype = dtype
        self._owner = owner

    # -- constructors (UnifiedTensor::new / ::empty, lib.rs:115-160) --------
    @classmethod
    def empty(cls, ctx: WgpuContext, shape: Sequence[int], dtype: DType = DType.FP32) -> "UnifiedTensor":
        nbytes = _prod(shape) * dtype.itemsize
        p = ctypes.c_void_p()
        call("rq_alloc", ctx.handle, nbytes, ctypes.byref(p))
        return cls(ctx, p.value or 0, shape, dtype)

    @classmethod
    def new(cls, ctx: WgpuContext, data, shape: Sequence[int] | None = None,
            dtype: DType | None = None) -> "UnifiedTensor":
        arr = np.asarray(data)
        if dtype is None:
            dtype = _INFERRED.get(arr.dtype.type, DType.FP32)
        arr = np.ascontiguousarray(arr, dtype=dtype.np)
        shape = tuple(arr.shape) if shape is None else tuple(shape)
        if _prod(shape) != arr.size:
            raise ValueError(f"shape {shape} does not match {arr.size} elements")
        t = cls.empty(ctx, shape, dtype)
        if arr.nbytes:
            call("rq_memcpy_h2d", ctx.handle, t.ptr, arr.ctypes.data, arr.nbytes, None)
        return t

    @property
    def numel(self) -> int:
        return math.prod(self.shape)

    @property
    def nbytes(self) -> int:
        return self.numel * self.dtype.itemsize

    def reshaped(self, shape: Sequence[int]) -> "UnifiedTensor":
        """Aliases the buffer with a new shape (lib.rs:198-213)."""
        if _prod(shape) != self.numel:
            raise ValueError("reshape changes the element count")
        v = UnifiedTensor(self.ctx, self.ptr, shape, self.dtype, owner=False)
        v._base = self
        return v

    def to_vec(self, ctx: WgpuContext | None = None) -> np.ndarray:
        """Waits for queued work and reads the buffer back (lib.rs:215-240)."""
        ctx = ctx or self.ctx
        out = np.empty(self.shape, dtype=self.dtype.np)
        if out.nbytes:
            call("rq_memcpy_d2h", ctx.handle, out.ctypes.data, self.ptr, out.nbytes, None)
        return out

    def zero_(self) -> "UnifiedTensor":
        call("rq_memset", self.ctx.handle, self.ptr, 0, self.nbytes, None)
        return self

    def __del__(self):
        try:
            if self._owner and self.ptr and self.ctx.handle:
                call("rq_free", self.ctx.handle, self.ptr)
        except Exception:
            pass
        self.ptr = 0


@dataclass
class QuantizedTensor:
    """A quantized Linear weight W[n_out, k_in] on the device.

    The reference has no quantized tensor type: ``upload_quantized``
    (rusty-loader/src/lib.rs:155-218) keeps codes/scales/biases as raw
    buffers only long enough to dequantize them to f32.  Here they stay
    quantized and feed the fused kernels."""

    codes: UnifiedTensor
    scales: UnifiedTensor
    biases: UnifiedTensor | None
    n_out: int
    k_in: int
    format: int
    group: int
    prep: UnifiedTensor | None = None  # affine: the prefill GEMM's scale table (rq_qweight_prepare)

    @classmethod
    def rowwise(cls, ctx: WgpuContext, q: np.ndarray, scales: np.ndarray) -> "QuantizedTensor":
        """Signed int8 codes ``q[n_out, k_in]`` and one f32 scale per row."""
        q = np.ascontiguousarray(q, dtype=np.int8)
        n, k = q.shape
        s = np.ascontiguousarray(scales, dtype=np.float32).reshape(n)
        return cls(UnifiedTensor.new(ctx, q, dtype=DType.I8), UnifiedTensor.new(ctx, s, dtype=DType.FP32),
                   None, n, k, _lib.RQ_Q_ROWWISE_I8, 0)

    @classmethod
    def from_rowwise(cls, codes: UnifiedTensor, scales: UnifiedTensor) -> "QuantizedTensor":
        """The same from device tensors: I8 [n_out, k_in] and FP32 [n_out]."""
        if codes.dtype is not DType.I8 or scales.dtype is not DType.FP32 or len(codes.shape) != 2:
            raise ValueError("codes must be I8 [n_out, k_in], scales FP32")
        n, k = codes.shape
        if scales.numel != n:
            raise ValueError(f"{n}x{k} weight needs {n} scales")
        return cls(codes, scales, None, n, k, _lib.RQ_Q_ROWWISE_I8, 0)

    @classmethod
    def affine(cls, ctx: WgpuContext, u: np.ndarray, scales: np.ndarray, biases: np.ndarray | None,
               group: int = 64, prepare: bool = True) -> "QuantizedTensor":
        """The reference's affine format: unsigned codes ``u[n_out, k_in]``,
        f32 scale and bias per ``group`` consecutive flat elements.  With
        ``prepare`` the prefill GEMM's scale table is built once here (load
        time, as upload_quantized does its one-time work), so no GEMM call
        rebuilds it."""
        u = np.ascontiguousarray(u, dtype=np.uint8)
        n, k = u.shape
        s = UnifiedTensor.new(ctx, np.ascontiguousarray(scales, dtype=np.float32).ravel(), dtype=DType.FP32)
        b = None if biases is None else UnifiedTensor.new(
            ctx, np.ascontiguousarray(biases, dtype=np.float32).ravel(), dtype=DType.FP32)
        need = -(-n * k // group)
        if s.numel < need or (b is not None and b.numel < need):
            raise ValueError(f"{n}x{k} weight with group {group} needs {need} scales/biases")
        qt = cls(UnifiedTensor.new(ctx, u, dtype=DType.U8), s, b, n, k, _lib.RQ_Q_AFFINE_U8, group)
        if prepare:
            qt.prepare(ctx)
        return qt

    @classmethod
    def from_affine(cls, codes: UnifiedTensor, scales: UnifiedTensor, biases: UnifiedTensor | None,
                    group: int = 64) -> "QuantizedTensor":
        """The same from device tensors: U8 [n_out, k_in], f32 scales and biases of
        consecutive groups (:meth:`prepare` builds the prefill GEMM's table)."""
        if codes.dtype is not DType.U8 or len(codes.shape) != 2 or scales.dtype is not DType.FP32 \
                or (biases is not None and biases.dtype is not DType.FP32):
            raise ValueError("codes must be U8 [n_out, k_in], scales and biases FP32")
        n, k = codes.shape
        need = -(-n * k // group) if group > 0 else 0
        if group <= 0 or scales.numel < need or (biases is not None and biases.numel < need):
            raise ValueError(f"{n}x{k} weight with group {group} needs {need} scales/biases")
        return cls(codes, scales, biases, n, k, _lib.RQ_Q_AFFINE_U8, group)

    @classmethod
    def affine4(cls, ctx: WgpuContext, u: np.ndarray, scales: np.ndarray, biases: np.ndarray | None,
                group: int = 64) -> "QuantizedTensor":
        """4-bit affine codes ``u[n_out, k_in]`` (values 0..15, one per array
        element here; two per byte on the device), f32 scale and bias per
        ``group`` elements of a row: RQ_Q_AFFINE_U4."""
        u = np.asarray(u)
        n, k = u.shape
        if k % 2 or group <= 0 or k % group:
            raise ValueError(f"k_in {k} must be even and a multiple of group {group}")
        if u.size and (u.min() < 0 or u.max() > 15):
            raise ValueError("4-bit codes are 0..15")
        u = u.astype(np.uint8)
        packed = UnifiedTensor.new(ctx, u[:, 0::2] | (u[:, 1::2] << 4), dtype=DType.U8)
        dev = lambda a: UnifiedTensor.new(  # noqa: E731
            ctx, np.ascontiguousarray(a, dtype=np.float32).reshape(n, -1), dtype=DType.FP32)
        return cls.from_affine4(packed, dev(scales), None if biases is None else dev(biases), group)

    @classmethod
    def from_affine4(cls, codes: UnifiedTensor, scales: UnifiedTensor, biases: UnifiedTensor | None,
                     group: int = 64) -> "QuantizedTensor":
        """The same from device tensors: packed codes U8 [n_out, k_in / 2] (the
        even element in the low nibble), scales and biases f32 with
        k_in / group values per row."""
        n, k = codes.shape[0], 2 * codes.shape[1]
        if codes.dtype is not DType.U8 or scales.dtype is not DType.FP32 \
                or (biases is not None and biases.dtype is not DType.FP32):
            raise ValueError("4-bit weight: codes must be U8, scales and biases FP32")
        if group <= 0 or k % group:
            raise ValueError(f"k_in {k} must be a multiple of group {group}")
        need = n * (k // group)
        if scales.numel != need or (biases is not None and biases.numel != need):
            raise ValueError(f"{n}x{k} weight with group {group} needs {need} scales/biases")
        return cls(codes, scales, biases, n, k, _lib.RQ_Q_AFFINE_U4, group)

    def prepare(self, ctx: WgpuContext, stream=None) -> None:
        """Builds the prefill GEMM's scale table of an affine weight
        (rq_qweight_prepare); nothing for weights that need none."""
        d = self.descriptor()
        d.prep = None
        nbytes = int(_lib.lib().rq_qweight_prep_bytes(ctypes.byref(d)))
        if nbytes == 0:
            self.prep = None
            return
        table = UnifiedTensor.empty(ctx, [nbytes // 4], DType.FP32)
        call("rq_qweight_prepare", ctx.handle, ctypes.byref(d), table.ptr, nbytes, _stream(stream))
        self.prep = table

    def dx_table(self, ctx: WgpuContext, stream=None) -> "UnifiedTensor | None":
        """The transposed-code table of the matrix-core input gradient
        (rq_qweight_dx_table), built on first use and kept with the weight;
        None when the weight is not served (see rq_qweight_dx_table_bytes)."""
        if getattr(self, "_dxt", None) is None:
            d = self.descriptor()
            nbytes = int(_lib.lib().rq_qweight_dx_table_bytes(ctypes.byref(d)))
            if nbytes == 0:
                return None
            table = UnifiedTensor.empty(ctx, [nbytes], DType.U8)
            call("rq_qweight_dx_table", ctx.handle, ctypes.byref(d), table.ptr, nbytes, _stream(stream))
            self._dxt = table
        return self._dxt

    def descriptor(self) -> rq_qweight:
        return rq_qweight(self.codes.ptr, self.scales.ptr, self.biases.ptr if self.biases is not None else None,
                          self.n_out, self.k_in, self.format, self.group,
                          self.prep.ptr if self.prep is not None else None)


class Rope:
    """How rotary positions turn a head: the frequencies on the device, and what
    of the head they turn (rq_rope, rq_rope_config).

    ``layout`` "half" pairs (i, i + rot_dim / 2) as the reference does,
    "interleaved" (2 i, 2 i + 1).  ``scaling`` for contexts ``factor`` times the
    ``trained`` one: "none", "linear", "stretch", "bands" or "ramp" (the last two
    with ``low`` and ``high`` turns within the trained context).  ``frequencies``
    (radians per position, rot_dim / 2 values) in place of all that."""

    LAYOUTS = {"half": _lib.RQ_ROPE_HALF, "interleaved": _lib.RQ_ROPE_INTERLEAVED}
    SCALINGS = {"none": _lib.RQ_ROPE_PLAIN, "linear": _lib.RQ_ROPE_LINEAR, "stretch": _lib.RQ_ROPE_STRETCH,
                "bands": _lib.RQ_ROPE_BANDS, "ramp": _lib.RQ_ROPE_RAMP}

    def __init__(self, ctx: WgpuContext, head_dim: int, rot_dim: int | None = None, layout: str = "half",
                 theta: float = 10000.0, scaling: str = "none", factor: float = 1.0, trained: float = 0.0,
                 low: float = 1.0, high: float = 32.0, frequencies=None, magnitude: float | None = None):
        rot_dim = head_dim if rot_dim is None else rot_dim
        if layout not in self.LAYOUTS or scaling not in self.SCALINGS:
            raise ValueError(f"layout {layout!r} / scaling {scaling!r}: expected one of {list(self.LAYOUTS)} / "
                             f"{list(self.SCALINGS)}")
        if frequencies is None:
            frequencies, own = self.frequencies_of(rot_dim, theta, scaling, factor, trained, low, high)
        else:
            frequencies, own = np.ascontiguousarray(frequencies, dtype=np.float64), 1.0
            if frequencies.shape != (rot_dim // 2,):
                raise ValueError(f"rot_dim {rot_dim} has {rot_dim // 2} frequencies")
        self.frequencies = UnifiedTensor.new(ctx, frequencies, dtype=DType.FP64)
        self.head_dim, self.rot_dim = head_dim, rot_dim
        self.descriptor = _lib.rq_rope(self.frequencies.ptr, head_dim, rot_dim, self.LAYOUTS[layout],
                                       own if magnitude is None else magnitude)

    @classmethod
    def frequencies_of(cls, rot_dim: int, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       trained: float = 0.0, low: float = 1.0, high: float = 32.0) -> tuple[np.ndarray, float]:
        """(frequencies, magnitude) of rq_rope_frequencies."""
        c = _lib.rq_rope_config(theta, factor, trained, low, high, cls.SCALINGS[scaling], rot_dim)
        f = (ctypes.c_double * max(rot_dim // 2, 1))()
        m = ctypes.c_float()
        call("rq_rope_frequencies", ctypes.byref(c), f, ctypes.byref(m))
        return np.array(f[:], dtype=np.float64), m.value


class PagedCache:
    """Keys and values of many sequences in pages (rq_kv_pages): ``k`` and ``v``
    [n_pages, n_kv_heads, page_size, head_dim] (``order`` "heads") or
    [n_pages, page_size, n_kv_heads, head_dim] ("positions"), ``table`` I32
    [n_seqs, max_pages]: the page of each sequence's positions p with p / page_size
    the column, -1 where there is none.  ``strides``: elements between pages, heads
    and positions where they are laid out otherwise."""

    def __init__(self, k: UnifiedTensor, v: UnifiedTensor, table: UnifiedTensor, order: str = "heads",
                 strides: Sequence[int] | None = None):
        if order not in ("heads", "positions"):
            raise ValueError(f"order {order!r}: expected 'heads' or 'positions'")
        if len(k.shape) != 4 or k.shape != v.shape or k.dtype is not v.dtype or len(table.shape) != 2 \
                or table.dtype is not DType.I32:
            raise ValueError(f"k {k.shape} / v {v.shape}: expected [n_pages, heads, positions, dim] of one type; table "
                             f"{table.shape}: expected I32 [n_seqs, max_pages]")
        self.k, self.v, self.table, self.dtype = k, v, table, k.dtype
        n_pages, a, b, self.head_dim = k.shape
        self.n_kv, page = (a, b) if order == "heads" else (b, a)
        if strides is None:
            strides = (0, 0, 0) if order == "heads" else (page * self.n_kv * self.head_dim, self.head_dim,
                                                          self.n_kv * self.head_dim)
        self.n_seqs, max_pages = table.shape
        self.descriptor = _lib.rq_kv_pages(k.ptr, v.ptr, table.ptr, *strides, 0, self.n_seqs, max_pages, n_pages, page)


class LoraSet:
    """Adapters of one Linear, for rows that each name one (rq_lora_set): ``a``
    [n_adapters, rank, k_in] (the reference's A transposed) and ``b`` [n_adapters,
    rank, n_out], both FP16 or both FP32, ``factors`` FP32 [n_adapters] (alpha / rank; None:
    1), ``ranks`` I32 [n_adapters] where some have fewer rows than ``rank``."""

    def __init__(self, a: UnifiedTensor, b: UnifiedTensor, factors: UnifiedTensor | None = None,
                 ranks: UnifiedTensor | None = None):
        if len(a.shape) != 3 or len(b.shape) != 3 or a.shape[:2] != b.shape[:2] or a.dtype not in _XDT \
                or b.dtype is not a.dtype:
            raise ValueError(f"a {a.shape} / b {b.shape}: expected [n_adapters, rank, k_in] and [n_adapters, rank, n_out] "
                             "of one type")
        n = a.shape[0]
        if (factors is not None and (factors.dtype is not DType.FP32 or factors.numel != n)) \
                or (ranks is not None and (ranks.dtype is not DType.I32 or ranks.numel != n)):
            raise ValueError("factors FP32 [n_adapters] and ranks I32 [n_adapters] do not match")
        self.a, self.b, self.factors, self.ranks = a, b, factors, ranks
        self.descriptor = _lib.rq_lora_set(a.ptr, b.ptr, factors.ptr if factors is not None else None,
                                           ranks.ptr if ranks is not None else None, n, a.shape[1], _XDT[a.dtype], 0)

    @classmethod
    def stack(cls, ctx: WgpuContext, adapters, factors=None, dtype: DType = DType.FP16) -> "LoraSet":
        """From host arrays as the reference holds them: pairs (A [k_in, rank],
        B [rank, n_out]), whose ranks may differ."""
        ranks = [a.shape[1] for a, _ in adapters]
        k, n, rank = adapters[0][0].shape[0], adapters[0][1].shape[1], max(max(ranks), 1)
        a = np.zeros((len(adapters), rank, k), dtype.np)
        b = np.zeros((len(adapters), rank, n), dtype.np)
        for i, (x, y) in enumerate(adapters):
            if x.shape != (k, ranks[i]) or y.shape != (ranks[i], n):
                raise ValueError(f"adapter {i}: A {x.shape} / B {y.shape} do not match [{k}, rank] / [rank, {n}]")
            a[i, :ranks[i]], b[i, :ranks[i]] = x.T, y
        T = lambda v, d: UnifiedTensor.new(ctx, v, dtype=d)  # noqa: E731
        return cls(T(a, dtype), T(b, dtype), None if factors is None else T(factors, DType.FP32),
                   T(ranks, DType.I32) if min(ranks) < rank else None)


_XDT = {DType.FP32: _lib.RQ_F32, DType.FP16: _lib.RQ_F16}


def _stream(stream):
    return None if stream is None else ctypes.c_void_p(stream if isinstance(stream, int) else stream.value)


class ComputeEngine:
    """Op surface of ``ComputeEngine`` (rusty-backend/src/lib.rs) for the
    quantized-linear path.  Every method enqueues work and returns."""

    def __init__(self, ctx: WgpuContext):
        self.ctx = ctx

    # ---- dequantization ---------------------------------------------------
    def dequantize(self, ctx: WgpuContext, input: UnifiedTensor, out: UnifiedTensor, stream=None) -> None:
        """lib.rs:4872-4899: ``out[4i+j] = byte j of input word i`` (unsigned,
        little-endian, no scale), for every input word that fits ``out``."""
        n_words = input.nbytes // 4
        call("rq_dequantize", ctx.handle, input.ptr, n_words, out.ptr, out.numel, _stream(stream))

    def affine_dequantize(self, ctx: WgpuContext, weight: UnifiedTensor, scales: UnifiedTensor,
                          biases: UnifiedTensor, out: UnifiedTensor, group: int = 64, fma: bool = False,
                          stream=None) -> None:
        """lib.rs:4939-4990: ``out[i] = f32(byte_i) * scales[i/64] + biases[i/64]``
        for every element of ``out`` (the reference's kernel hard-codes 64)."""
        n_groups = min(scales.numel, biases.numel if biases is not None else scales.numel)
        call("rq_affine_dequantize", ctx.handle, weight.ptr, weight.nbytes // 4, scales.ptr,
             biases.ptr if biases is not None else None, n_groups, out.ptr, out.numel, group,
             _lib.RQ_AFFINE_FMA if fma else 0, _stream(stream))

    def dequantize_weight(self, ctx: WgpuContext, w: QuantizedTensor, out: UnifiedTensor, stream=None) -> None:
        """Load-time dequantization of a QuantizedTensor to f32 [n_out, k_in]."""
        if out.numel != w.n_out * w.k_in:
            raise ValueError("output size does not match the weight")
        d = w.descriptor()
        call("rq_qweight_dequantize", ctx.handle, ctypes.byref(d), out.ptr, _stream(stream))

    # ---- f32 matmul family -----------------------------------------------
    def matmul(self, ctx: WgpuContext, a: UnifiedTensor, b: UnifiedTensor, out: UnifiedTensor,
               stream=None) -> None:
        """lib.rs:4403-4453: m, k, n = a.shape[0], a.shape[1], b.shape[1]."""
        m, k, n = a.shape[0], a.shape[1], b.shape[1]
        self._check_mm(a, b, out, (m, k), (k, n), (m, n))
        call("rq_matmul", ctx.handle, a.ptr, b.ptr, out.ptr, m, k, n, _stream(stream))

    def matmul_bt(self, ctx: WgpuContext, a: UnifiedTensor, b: UnifiedTensor, out: UnifiedTensor,
                  stream=None) -> None:
        """lib.rs:4299-4349: m, k, n = a.shape[0], a.shape[1], b.shape[0]."""
        m, k, n = a.shape[0], a.shape[1], b.shape[0]
        self._check_mm(a, b, out, (m, k), (n, k), (m, n))
        call("rq_matmul_bt", ctx.handle, a.ptr, b.ptr, out.ptr, m, k, n, _stream(stream))

    def matmul_at(self, ctx: WgpuContext, a: UnifiedTensor, b: UnifiedTensor, out: UnifiedTensor,
                  stream=None) -> None:
        """lib.rs:4351-4401: m, k, n = a.shape[1], a.shape[0], b.shape[1]."""
        m, k, n = a.shape[1], a.shape[0], b.shape[1]
        self._check_mm(a, b, out, (k, m), (k, n), (m, n))
        call("rq_matmul_at", ctx.handle, a.ptr, b.ptr, out.ptr, m, k, n, _stream(stream))

    @staticmethod
    def _check_mm(a, b, out, sa, sb, so):
        for t, s, nm in ((a, sa, "a"), (b, sb, "b"), (out, so, "out")):
            if t.dtype is not DType.FP32 or t.numel != _prod(s):
                raise ValueError(f"{nm}: expected f32 with {_prod(s)} elements for shape {s}, "
                                 f"got {t.dtype.name} {t.shape}")

    # ---- fused quantized linear -------------------------------------------
    def qmatmul(self, ctx: WgpuContext, x: UnifiedTensor, w: QuantizedTensor, out: UnifiedTensor,
                stream=None) -> None:
        """``out[m, n_out] = x[m, k_in] . deq(w)^T`` with dequantization fused
        into the product (what ``Linear::forward``, rusty-graph/src/lib.rs:69,
        computes on the reference's dequantized weight)."""
        if x.dtype not in _XDT or out.dtype not in _XDT:
            raise ValueError("x and out must be FP16 or FP32")
        m = x.numel // w.k_in if w.k_in else x.shape[0]
        if x.numel != m * w.k_in or out.numel != m * w.n_out:
            raise ValueError(f"x {x.shape} / out {out.shape} do not match weight [{w.n_out}, {w.k_in}]")
        d = w.descriptor()
        call("rq_qmatmul", ctx.handle, ctypes.byref(d), x.ptr, _XDT[x.dtype], out.ptr, _XDT[out.dtype], m,
             _stream(stream))

    def qmatmul_lora(self, ctx: WgpuContext, x: UnifiedTensor, w: QuantizedTensor, lora_a: UnifiedTensor,
                     lora_b: UnifiedTensor, out: UnifiedTensor, workspace: UnifiedTensor | None = None,
                     stream=None, tree: bool = False) -> None:
        """``Linear::forward`` with a LoRA adapter (rusty-graph/src/lib.rs:69-83):
        ``out = x . deq(w)^T + (x . A) . B``, A f32 [k_in, rank], B f32
        [rank, n_out], unscaled as the reference adds it.  ``tree``: x . A as
        a fixed-order reduction tree (rq_qmatmul_lora_ex, RQ_LORA_TREE) instead
        of the reference's k-ascending chain -- within f32 rounding of it, not
        its bits, and without the chain's k_in-step latency."""
        if x.dtype not in _XDT or out.dtype not in _XDT:
            raise ValueError("x and out must be FP16 or FP32")
        if lora_a.dtype is not DType.FP32 or lora_b.dtype is not DType.FP32:
            raise ValueError("the adapter's A and B must be FP32")
        m = x.numel // w.k_in if w.k_in else x.shape[0]
        rank = lora_a.numel // w.k_in if w.k_in else 0
        if x.numel != m * w.k_in or out.numel != m * w.n_out or lora_a.numel != w.k_in * rank \
                or lora_b.numel != rank * w.n_out:
            raise ValueError(f"x {x.shape} / A {lora_a.shape} / B {lora_b.shape} / out {out.shape} do not match "
                             f"weight [{w.n_out}, {w.k_in}]")
        flags = _lib.RQ_LORA_TREE if tree else 0
        need = _lib.lib().rq_qmatmul_lora_ex_workspace(m, w.k_in, w.n_out, rank, _XDT[x.dtype], _XDT[out.dtype],
                                                       flags)
        if workspace is None:
            workspace = UnifiedTensor.empty(ctx, [max(need, 1)], DType.U8)
        d = w.descriptor()
        if tree:
            call("rq_qmatmul_lora_ex", ctx.handle, ctypes.byref(d), x.ptr, _XDT[x.dtype], lora_a.ptr, lora_b.ptr,
                 rank, out.ptr, _XDT[out.dtype], m, flags, workspace.ptr, workspace.numel * workspace.dtype.itemsize,
                 _stream(stream))
        else:
            call("rq_qmatmul_lora", ctx.handle, ctypes.byref(d), x.ptr, _XDT[x.dtype], lora_a.ptr, lora_b.ptr, rank,
                 out.ptr, _XDT[out.dtype], m, workspace.ptr, workspace.numel * workspace.dtype.itemsize,
                 _stream(stream))

    def qmatmul_loras(self, ctx: WgpuContext, x: UnifiedTensor, w: QuantizedTensor, adapters: LoraSet,
                      ids: UnifiedTensor, out: UnifiedTensor, workspace: UnifiedTensor | None = None,
                      stream=None) -> None:
        """``out[t] = x[t] . deq(w)^T + factors[i] (x[t] . A_i^T) . B_i`` with i =
        ``ids[t]`` (I32 [m] on the device; none for i < 0): a batch of tokens of many
        requests, each with its own adapter (rq_qmatmul_loras).  Without a
        ``workspace`` the call allocates one; a captured call is given its own,
        which lives as long as the graph."""
        m = self._check_loras(x, w, adapters, out)
        if ids.dtype is not DType.I32 or ids.numel != m:
            raise ValueError(f"ids must be I32 [{m}]")
        if workspace is None:
            workspace = self.qmatmul_loras_workspace(ctx, x, w, adapters, out)
        d = w.descriptor()
        call("rq_qmatmul_loras", ctx.handle, ctypes.byref(d), ctypes.byref(adapters.descriptor), ids.ptr, x.ptr,
             _XDT[x.dtype], out.ptr, _XDT[out.dtype], m, workspace.ptr, workspace.nbytes, _stream(stream))

    def qmatmul_loras_workspace(self, ctx: WgpuContext, x: UnifiedTensor, w: QuantizedTensor, adapters: LoraSet,
                                out: UnifiedTensor) -> UnifiedTensor:
        """A workspace for ``qmatmul_loras`` calls of these shapes (one per call in flight)."""
        m = self._check_loras(x, w, adapters, out)
        need = int(_lib.lib().rq_qmatmul_loras_workspace(ctypes.byref(adapters.descriptor), m, w.k_in, w.n_out,
                                                         _XDT[x.dtype], _XDT[out.dtype]))
        return UnifiedTensor.empty(ctx, [max(need, 1)], DType.U8)

    @staticmethod
    def _check_loras(x, w, adapters, out) -> int:
        if x.dtype not in _XDT or out.dtype not in _XDT:
            raise ValueError("x and out must be FP16 or FP32")
        n = x.numel
        m = n // w.k_in if w.k_in else x.shape[0]
        if n != m * w.k_in or out.numel != m * w.n_out or adapters.a.shape[2] != w.k_in \
                or adapters.b.shape[2] != w.n_out:
            raise ValueError(f"x {x.shape} / A {adapters.a.shape} / B {adapters.b.shape} / out {out.shape} do not match "
                             f"weight [{w.n_out}, {w.k_in}]")
        return m

    def qmatmul_dx(self, ctx: WgpuContext, dy: UnifiedTensor, w: QuantizedTensor, dx: UnifiedTensor,
                   stream=None, mfma: bool = False, workspace: UnifiedTensor | None = None) -> None:
        """Input gradient of ``qmatmul`` with the weight frozen:
        ``dx[m, k_in] = dy[m, n_out] . deq(w)`` -- the ``grad_a`` of
        ``MatMulNode::backward`` (rusty-autograd/src/lib.rs:152-158).
        ``mfma``: on the matrix cores (rq_qmatmul_dx_mfma, per-row int8
        weights; the weight's transposed table is built on first use) -- the
        f32 bar, not the f32 chain's bit pattern."""
        if dy.dtype not in _XDT or dx.dtype not in _XDT:
            raise ValueError("dy and dx must be FP16 or FP32")
        m = dy.numel // w.n_out if w.n_out else dx.shape[0]
        if dy.numel != m * w.n_out or dx.numel != m * w.k_in:
            raise ValueError(f"dy {dy.shape} / dx {dx.shape} do not match weight [{w.n_out}, {w.k_in}]")
        d = w.descriptor()
        if not mfma:
            call("rq_qmatmul_dx", ctx.handle, ctypes.byref(d), dy.ptr, _XDT[dy.dtype], dx.ptr, _XDT[dx.dtype], m,
                 _stream(stream))
            return
        table = w.dx_table(ctx, stream)
        if table is None:
            raise ValueError(f"weight [{w.n_out}, {w.k_in}] is not served by the matrix-core input gradient")
        need = int(_lib.lib().rq_qmatmul_dx_mfma_workspace(m, w.n_out))
        if workspace is None:
            workspace = UnifiedTensor.empty(ctx, [max(need, 1)], DType.U8)
        call("rq_qmatmul_dx_mfma", ctx.handle, ctypes.byref(d), table.ptr, dy.ptr, _XDT[dy.dtype], dx.ptr,
             _XDT[dx.dtype], m, workspace.ptr, workspace.numel * workspace.dtype.itemsize, _stream(stream))

    def mlp_swiglu(self, ctx: WgpuContext, x: UnifiedTensor, gate: QuantizedTensor, up: QuantizedTensor,
                   down: QuantizedTensor, out: UnifiedTensor, h: UnifiedTensor | None = None,
                   stream=None) -> UnifiedTensor:
        """``MLP::forward`` (rusty-graph/src/lib.rs:317-323):
        ``out = down(silu(x . gate^T) * (x . up^T))``.  ``h`` is the fp16
        workspace (2 * m * I values); returned, its first m*I hold silu(g)*u."""
        m = x.numel // gate.k_in if gate.k_in else out.shape[0]
        if h is None:
            h = UnifiedTensor.empty(ctx, [2, m, gate.n_out], DType.FP16)
        if h.dtype is not DType.FP16 or h.numel < 2 * m * gate.n_out:
            raise ValueError("h must be an fp16 workspace of 2*m*I values")
        if out.numel != m * down.n_out:
            raise ValueError("out does not match [m, H]")
        dg, du, dd = gate.descriptor(), up.descriptor(), down.descriptor()
        call("rq_mlp_swiglu", ctx.handle, ctypes.byref(dg), ctypes.byref(du), ctypes.byref(dd), x.ptr,
             _XDT[x.dtype], h.ptr, out.ptr, _XDT[out.dtype], m, _stream(stream))
        return h

    # ---- attention ----------------------------------------------------------
    def attn_packed(self, ctx: WgpuContext, q: UnifiedTensor, k: UnifiedTensor, v: UnifiedTensor,
                    starts: UnifiedTensor, out: UnifiedTensor, scale: float | None = None, q_row: int | None = None,
                    k_row: int | None = None, v_row: int | None = None, out_row: int | None = None,
                    stream=None) -> None:
        """Causal GQA attention over packed prompts (rq_attn_packed): q and out
        [tokens, n_heads, head_dim], k and v [tokens, n_kv_heads, head_dim],
        ``starts`` I32 [n_seqs + 1] on the device.  ``*_row``: elements between
        the rows of consecutive tokens where they are not packed (q, k and v in
        the rows of one fused q/k/v product)."""
        if len(q.shape) != 3 or len(k.shape) != 3 or k.shape != v.shape or out.shape != q.shape \
                or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
            raise ValueError(f"q {q.shape} / k {k.shape} / v {v.shape} / out {out.shape}: expected [tokens, heads, dim]")
        a = _attn(q, k, v, out, k.shape[1], scale)
        a.q_row, a.k_row, a.v_row, a.out_row = q_row or 0, k_row or 0, v_row or 0, out_row or 0
        if starts.dtype is not DType.I32 or starts.numel < 1:
            raise ValueError("starts must be I32 [n_seqs + 1]")
        call("rq_attn_packed", ctx.handle, ctypes.byref(a), q.ptr, k.ptr, v.ptr, starts.ptr, starts.numel - 1,
             q.shape[0], out.ptr, _stream(stream))

    def attn_tree(self, ctx: WgpuContext, q: UnifiedTensor, k: UnifiedTensor, v: UnifiedTensor,
                  starts: UnifiedTensor, lengths: UnifiedTensor, mask: UnifiedTensor | None, out: UnifiedTensor,
                  max_nodes: int, scale: float | None = None, workspace: UnifiedTensor | None = None,
                  q_row: int | None = None, out_row: int | None = None, strides: Sequence[int] | None = None,
                  stream=None) -> None:
        """Attention of drafted tokens over a KV cache (rq_attn_tree): q and out
        [tokens, n_heads, head_dim], the cache k and v [n_seqs, n_kv_heads,
        capacity, head_dim] (``strides``: elements between sequences, heads and
        positions where it is laid out otherwise), ``starts`` I32 [n_seqs + 1],
        ``lengths`` I32 [n_seqs], ``mask`` U64 [tokens] or None (chains).
        Without a ``workspace`` the call allocates one where it needs it; a
        captured call is given its own, which lives as long as the graph."""
        if len(q.shape) != 3 or len(k.shape) != 4 or k.shape != v.shape or out.shape != q.shape \
                or k.shape[3] != q.shape[2]:
            raise ValueError(f"q {q.shape} / out {out.shape}: expected [tokens, heads, dim]; k {k.shape} / v {v.shape}: "
                             "expected [n_seqs, kv heads, capacity, dim]")
        n_seqs, n_kv, capacity, _ = k.shape
        if starts.dtype is not DType.I32 or starts.numel != n_seqs + 1 or lengths.dtype is not DType.I32 \
                or lengths.numel != n_seqs or (mask is not None and (mask.dtype is not DType.U64
                                                                    or mask.numel != q.shape[0])):
            raise ValueError("starts I32 [n_seqs + 1], lengths I32 [n_seqs] and mask U64 [tokens] do not match")
        a = _attn(q, k, v, out, n_kv, scale)
        a.q_row, a.out_row = q_row or 0, out_row or 0
        ss, sh, sp = strides or (0, 0, 0)
        c = _lib.rq_kv_cache(k.ptr, v.ptr, ss, sh, sp, n_seqs, capacity)
        if workspace is None:
            workspace = self.attn_tree_workspace(ctx, q, k, max_nodes)
        call("rq_attn_tree", ctx.handle, ctypes.byref(a), ctypes.byref(c), q.ptr, starts.ptr, lengths.ptr,
             mask.ptr if mask is not None else None, q.shape[0], max_nodes, out.ptr, workspace.ptr, workspace.nbytes,
             _stream(stream))

    def attn_tree_workspace(self, ctx: WgpuContext, q: UnifiedTensor, k: UnifiedTensor,
                            max_nodes: int) -> UnifiedTensor:
        """A workspace for ``attn_tree`` calls of these shapes (one per call in flight)."""
        a = _attn(q, k, k, q, k.shape[1], None)
        need = int(_lib.lib().rq_attn_tree_workspace(ctypes.byref(a), k.shape[0], q.shape[0], max_nodes, k.shape[2]))
        return UnifiedTensor.empty(ctx, [max(need, 1)], DType.U8)


    # ---- rotary positions, paged caches ----------------------------------------
    def rope(self, ctx: WgpuContext, x: UnifiedTensor, rope: Rope, positions: UnifiedTensor,
             out: UnifiedTensor | None = None, backward: bool = False, x_row: int | None = None,
             out_row: int | None = None, stream=None) -> None:
        """``out = x`` [tokens, heads, head_dim] with each head turned by its token's
        position (kernels.wgsl:60-79, which has one position for all; rq_rope_rows), in
        place without ``out``.  ``positions`` I32 [tokens].  ``backward``: the gradient of
        x from that of out.  ``*_row``: elements between the rows of consecutive tokens."""
        if out is None:
            out, out_row = x, x_row
        if len(x.shape) != 3 or out.shape != x.shape or x.shape[2] != rope.head_dim or x.dtype not in _XDT \
                or out.dtype is not x.dtype:
            raise ValueError(f"x {x.shape} / out {out.shape}: expected [tokens, heads, {rope.head_dim}], FP16 or FP32")
        tokens, heads, _ = x.shape
        if positions.dtype is not DType.I32 or positions.numel != tokens:
            raise ValueError(f"positions must be I32 [{tokens}]")
        call("rq_rope_rows", ctx.handle, ctypes.byref(rope.descriptor), x.ptr, x_row or 0, positions.ptr, tokens, heads,
             _XDT[x.dtype], out.ptr, out_row or 0, _lib.RQ_ROPE_BACKWARD if backward else 0, _stream(stream))

    def rope_append(self, ctx: WgpuContext, q: UnifiedTensor, k: UnifiedTensor, v: UnifiedTensor, rope: Rope,
                    positions: UnifiedTensor, cache: PagedCache, out: UnifiedTensor, starts: UnifiedTensor | None = None,
                    q_row: int | None = None, k_row: int | None = None, v_row: int | None = None,
                    out_row: int | None = None, stream=None) -> None:
        """``out = q`` turned by position, ``k`` turned and ``v`` copied into the cache's
        pages (rq_rope_append): q and out [tokens, n_heads, dim], k and v
        [tokens, n_kv_heads, dim], ``positions`` I32 [tokens], each within its
        sequence.  ``starts`` I32 [n_seqs + 1]: sequence s is tokens starts[s] ..
        starts[s+1]-1; without, token t is all of sequence t."""
        if len(q.shape) != 3 or k.shape != (q.shape[0], cache.n_kv, cache.head_dim) or v.shape != k.shape \
                or out.shape != q.shape or q.shape[2] != cache.head_dim or cache.dtype is not q.dtype:
            raise ValueError(f"q {q.shape} / k {k.shape} / v {v.shape} / out {out.shape}: expected [tokens, heads, dim] of "
                             f"the cache's {cache.n_kv} heads of {cache.head_dim} and its type")
        tokens = q.shape[0]
        if positions.dtype is not DType.I32 or positions.numel != tokens or (
                starts is not None and (starts.dtype is not DType.I32 or starts.numel != cache.n_seqs + 1)):
            raise ValueError("positions I32 [tokens] and starts I32 [n_seqs + 1] do not match")
        a = _attn(q, k, v, out, cache.n_kv, None)
        a.q_row, a.k_row, a.v_row, a.out_row = q_row or 0, k_row or 0, v_row or 0, out_row or 0
        call("rq_rope_append", ctx.handle, ctypes.byref(rope.descriptor), ctypes.byref(a), ctypes.byref(cache.descriptor),
             q.ptr, k.ptr, v.ptr, starts.ptr if starts is not None else None, positions.ptr, tokens, out.ptr,
             _stream(stream))

    def attn_paged(self, ctx: WgpuContext, q: UnifiedTensor, cache: PagedCache, lengths: UnifiedTensor,
                   out: UnifiedTensor, scale: float | None = None, workspace: UnifiedTensor | None = None,
                   q_row: int | None = None, out_row: int | None = None, stream=None) -> None:
        """Attention of one new token per sequence over a paged cache
        (rq_attn_paged): q and out [n_seqs, n_heads, head_dim], ``lengths`` I32
        [n_seqs], the token itself included.  Without a ``workspace`` the call
        allocates one; a captured call is given its own, which lives as long as the
        graph."""
        if len(q.shape) != 3 or out.shape != q.shape or q.shape[0] != cache.n_seqs or q.shape[2] != cache.head_dim:
            raise ValueError(f"q {q.shape} / out {out.shape}: expected [{cache.n_seqs}, heads, {cache.head_dim}]")
        if lengths.dtype is not DType.I32 or lengths.numel != cache.n_seqs:
            raise ValueError(f"lengths must be I32 [{cache.n_seqs}]")
        a = _attn(q, cache.k, cache.v, out, cache.n_kv, scale)
        a.q_row, a.out_row = q_row or 0, out_row or 0
        if workspace is None:
            workspace = self.attn_paged_workspace(ctx, q, cache)
        call("rq_attn_paged", ctx.handle, ctypes.byref(a), ctypes.byref(cache.descriptor), q.ptr, lengths.ptr, out.ptr,
             workspace.ptr, workspace.nbytes, _stream(stream))

    def attn_paged_workspace(self, ctx: WgpuContext, q: UnifiedTensor, cache: PagedCache) -> UnifiedTensor:
        """A workspace for ``attn_paged`` calls of these shapes (one per call in flight)."""
        a = _attn(q, cache.k, cache.v, q, cache.n_kv, None)
        need = int(_lib.lib().rq_attn_paged_workspace(ctypes.byref(a), ctypes.byref(cache.descriptor)))
        return UnifiedTensor.empty(ctx, [max(need, 1)], DType.U8)


def _attn(q, k, v, out, n_kv, scale):
    if q.dtype not in _XDT or k.dtype is not q.dtype or v.dtype is not q.dtype or out.dtype is not q.dtype:
        raise ValueError("q, k, v and out must all be FP16 or all FP32")
    return _lib.rq_attn(q.shape[1], n_kv, q.shape[2], _XDT[q.dtype], 0.0 if scale is None else scale, 0, 0, 0, 0, 0)
