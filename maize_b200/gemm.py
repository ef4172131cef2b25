"""Host-side mirror of the reference's GEMM call shape over the C ABI.

The reference builds its GEMM from ``Matrix::new(ptr, nrows, ncols)`` pairs
(crates/maize_tile/src/gmem/matrix.rs:13-18, src/main.rs:46-48) handed to
``sm80_gemm_smem_multibuffer`` (crates/maize_tile/src/gemm/mod.rs:37-90).  The
same shape is kept: ``Matrix`` is {ptr, nrows, ncols}; ``Context.gemm`` takes A
(M x K), B (N x K, K-major) and C (M x N) and launches the sm_100a kernels.
torch is used only for device memory and streams.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

from . import _ffi


class MaizeError(RuntimeError):
    def __init__(self, status: int, message: str = ""):
        self.status = status
        name = _ffi.STATUS_NAMES.get(status, f"status {status}")
        super().__init__(f"{name}: {message}" if message else name)


@dataclass(frozen=True)
class Matrix:
    """{ptr, nrows, ncols} of a dense row-major bf16 matrix in device memory."""
    ptr: int
    nrows: int
    ncols: int

    @classmethod
    def new(cls, ptr: int, nrows: int, ncols: int) -> "Matrix":
        return cls(int(ptr), int(nrows), int(ncols))

    @classmethod
    def from_tensor(cls, t) -> "Matrix":
        import torch
        if t.dim() != 2 or t.dtype != torch.bfloat16 or not t.is_contiguous():
            raise MaizeError(_ffi.INVALID_ARG, "expected a contiguous 2-D bfloat16 tensor")
        return cls(t.data_ptr(), t.shape[0], t.shape[1])

    def as_c(self) -> _ffi.GlobalMatrix:
        return _ffi.GlobalMatrix(self.ptr, self.nrows, self.ncols)


def _stream_handle(stream) -> Optional[int]:
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


_torch = None
_raw_stream = None
_empty = None
_current_device = None
_devices = ()


def _types():
    """The torch module, imported with the first call that has tensors to look at; with it, torch's name of every device, and the
    shortest ways that this torch has to a device's current stream and to a new tensor on the current device."""
    global _torch, _raw_stream, _empty, _current_device, _devices
    if _torch is None:
        import torch
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda device: torch.cuda.current_stream(device).cuda_stream)
        # sizes, strides, type -> tensor of the current device: 0.75 us, torch.empty takes 1.6
        short = getattr(getattr(getattr(torch._C, "_dynamo", None), "guards", None), "_empty_strided_cuda", None)
        _empty = _on_trial(short) if short else None
        _current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
        _devices = tuple(torch.device("cuda", i) for i in range(torch.cuda.device_count()))
        _torch = torch
    return _torch


def _on_trial(short):
    """``short``, a way to a new tensor that torch does not document, for its first call: if it does not give what was asked for,
    this call and all later ones go by ``torch.empty``."""
    def first(shape, strides, dtype):
        global _empty
        try:
            t = short(shape, strides, dtype)
            right = t.shape == shape and t.stride() == strides and t.dtype is dtype and t.get_device() == _current_device()
        except _torch.cuda.OutOfMemoryError:
            raise
        except Exception:
            right = False
        _empty = short if right else None
        return t if right else _torch.empty(*shape, dtype=dtype, device=_devices[_current_device()])
    return first


class Context:
    """One per host thread / stream; owns the device status word and tunables."""

    def __init__(self, device: int = 0):
        self._lib = _ffi.load()
        handle = ctypes.c_void_p()
        st = self._lib.maize_ctx_create(int(device), ctypes.byref(handle))
        if st != _ffi.OK:
            raise MaizeError(st, self._lib.maize_status_string(st).decode())
        self._h = handle
        self._ctx = handle.value  # the same for the calls that do not go through ctypes
        self._calls = _ffi.load_calls()
        self.device = int(device)

    def close(self) -> None:
        if getattr(self, "_h", None):
            self._lib.maize_ctx_destroy(self._h)
            self._h = self._ctx = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    # ------------------------------------------------------------ helpers --
    def _check(self, st: int) -> None:
        if st != _ffi.OK:
            raise MaizeError(st, self._lib.maize_last_error(self._h).decode())

    def set(self, key: str, value: int) -> None:
        self._check(self._lib.maize_ctx_set(self._h, key.encode(), int(value)))

    def get(self, key: str) -> int:
        out = ctypes.c_int64()
        self._check(self._lib.maize_ctx_get(self._h, key.encode(), ctypes.byref(out)))
        return out.value

    @property
    def launch_count(self) -> int:
        return int(self._lib.maize_ctx_launch_count(self._h))

    def pick_kernel(self, m: int, n: int, k: int) -> str:
        return self._lib.maize_kernel_name(self._lib.maize_pick_kernel(self._h, m, n, k)).decode()

    @property
    def last_kernel(self) -> str:
        """Name of the GEMM kernel the last call on this context launched ("" before the first)."""
        kid = self.get("last_kernel")
        return self._lib.maize_kernel_name(kid).decode() if kid > 0 else ""

    def poll(self, stream=None) -> None:
        """Synchronise the stream and raise if a device wait timed out."""
        self._check(self._lib.maize_ctx_poll(self._h, _stream_handle(stream)))

    # --------------------------------------------------------------- GEMM --
    def gemm_matrices(self, a: Matrix, b: Matrix, c: Matrix, stream=None) -> None:
        """C = A @ B.T through the {ptr, nrows, ncols} bundles."""
        ca, cb, cc = a.as_c(), b.as_c(), c.as_c()
        self._check(self._lib.maize_gemm_bf16_m(self._h, ctypes.byref(ca), ctypes.byref(cb), ctypes.byref(cc),
                                                _stream_handle(stream)))

    def gemm_raw(self, a_ptr, a_rows, a_cols, b_ptr, b_rows, b_cols, c_ptr, c_rows, c_cols, stream=None) -> None:
        self._check(self._lib.maize_gemm_bf16(self._h, a_ptr, a_rows, a_cols, b_ptr, b_rows, b_cols, c_ptr, c_rows,
                                              c_cols, _stream_handle(stream)))

    def gemm_ld(self, a_ptr, lda, b_ptr, ldb, c_ptr, ldc, m, n, k, stream=None) -> None:
        self._check(self._lib.maize_gemm_bf16_ld(self._h, a_ptr, lda, b_ptr, ldb, c_ptr, ldc, m, n, k,
                                                 _stream_handle(stream)))

    def gemm_host(self, a_ptr, a_rows, a_cols, b_ptr, b_rows, b_cols, c_ptr, c_rows, c_cols, stream=None) -> None:
        """Host buffers in, host buffer out; copies and the wait are inside the call."""
        self._check(self._lib.maize_gemm_bf16_host(self._h, a_ptr, a_rows, a_cols, b_ptr, b_rows, b_cols, c_ptr,
                                                   c_rows, c_cols, _stream_handle(stream)))

    def gemm(self, a, b, out=None, stream=None):
        """``out = a @ b.T`` for bf16 CUDA tensors: a is M x K, b is N x K; rows may be strided."""
        import torch
        for name, t in (("a", a), ("b", b)):
            if t.dim() != 2 or t.dtype != torch.bfloat16 or not t.is_cuda or (t.shape[1] > 1 and t.stride(1) != 1):
                raise MaizeError(_ffi.INVALID_ARG, f"{name}: expected a 2-D bfloat16 CUDA tensor with unit column stride")
        m, k = a.shape
        n, kb = b.shape
        if k != kb:
            raise MaizeError(_ffi.INVALID_ARG, "a.shape[1] != b.shape[1] (b is stored N x K)")
        if out is None:
            out = torch.empty((m, n), dtype=torch.bfloat16, device=a.device)
        elif out.shape != (m, n) or out.dtype != torch.bfloat16 or not out.is_cuda or (n > 1 and out.stride(1) != 1):
            raise MaizeError(_ffi.INVALID_ARG, "out: expected an M x N bfloat16 CUDA tensor with unit column stride")
        lda = a.stride(0) if m > 1 else max(k, 1)
        ldb = b.stride(0) if n > 1 else max(k, 1)
        ldc = out.stride(0) if m > 1 else max(n, 1)
        self.gemm_ld(a.data_ptr(), lda, b.data_ptr(), ldb, out.data_ptr(), ldc, m, n, k, stream)
        return out

    def gemm_gated(self, a, b, out, rows_landed_ptr: int, landed_base: int, rows_per_count: int, stream=None):
        """``out = a @ b.T`` for an ``a`` whose rows are still arriving in row order: the kernel reads rows
        [0, r) only once the 32-bit word at ``rows_landed_ptr`` has reached landed_base + ceil(r / rows_per_count).
        The wait is bounded ("timeout_ns"); ``poll()`` reports a count that never came as a timeout."""
        m, k = a.shape
        n = b.shape[0]
        if b.shape[1] != k or tuple(out.shape) != (m, n):
            raise MaizeError(_ffi.INVALID_ARG, "gemm_gated: a is M x K, b is N x K, out is M x N")
        lda = a.stride(0) if m > 1 else max(k, 1)
        ldb = b.stride(0) if n > 1 else max(k, 1)
        ldc = out.stride(0) if m > 1 else max(n, 1)
        self._check(self._lib.maize_gemm_bf16_gated(self._h, a.data_ptr(), lda, b.data_ptr(), ldb, out.data_ptr(), ldc,
                                                    m, n, k, rows_landed_ptr, landed_base & 0xFFFFFFFF, rows_per_count,
                                                    _stream_handle(stream)))
        return out

    PROFILE_SLOTS = ("producer_wait_empty", "mma_wait_full", "mma_wait_acc_empty", "epilogue_wait_acc_full",
                     "epilogue_drain", "cta_cycles", "tiles", "spare")

    def read_profile(self, stream=None):
        """Per-CTA cycle counters of the last launch (after ``set("profile", 1)``): list of dicts."""
        buf = (ctypes.c_uint64 * (8 * 1024))()
        n = self._lib.maize_ctx_read_profile(self._h, buf, 1024, _stream_handle(stream))
        return [dict(zip(self.PROFILE_SLOTS, buf[8 * i:8 * i + 8])) for i in range(n)]

    # ------------------------------------------------- multi-GPU building blocks --
    def mc_push(self, src_ptr: int, mc_dst_ptr: int, nbytes: int, mc_flag_ptr: int, flag_value: int, ctas: int = 0,
                stream=None) -> None:
        """Push local bytes to every GPU's replica through the multicast address, then publish a flag value."""
        self._check(self._lib.maize_mc_push(self._h, src_ptr, mc_dst_ptr, nbytes, mc_flag_ptr, flag_value & 0xFFFFFFFF,
                                            ctas, _stream_handle(stream)))

    def mc_push_after(self, wait_flag_ptr: int, wait_value: int, src_ptr: int, mc_dst_ptr: int, nbytes: int,
                      mc_flag_ptr: int, flag_value: int, ctas: int = 0, stream=None) -> None:
        """Like mc_push, but the kernel first waits for the local word at wait_flag_ptr to reach wait_value."""
        self._check(self._lib.maize_mc_push_after(self._h, wait_flag_ptr, wait_value & 0xFFFFFFFF, src_ptr, mc_dst_ptr,
                                                  nbytes, mc_flag_ptr, flag_value & 0xFFFFFFFF, ctas,
                                                  _stream_handle(stream)))

    def scatter_push(self, src_ptr: int, peer_dst_ptrs, peer_flag_ptrs, root: int, nbytes: int, flag_value: int,
                     ctas: int = 0, stream=None) -> None:
        """Root: store chunk p of the source into rank p's landing buffer and publish a flag there."""
        world = len(peer_dst_ptrs)
        dst = (ctypes.c_void_p * world)(*[ctypes.c_void_p(int(x)) for x in peer_dst_ptrs])
        flg = (ctypes.c_void_p * world)(*[ctypes.c_void_p(int(x)) for x in peer_flag_ptrs])
        self._check(self._lib.maize_scatter_push(self._h, src_ptr, dst, flg, world, root, nbytes,
                                                 flag_value & 0xFFFFFFFF, ctas, _stream_handle(stream)))

    def copy_async(self, dst_ptr: int, src_ptr: int, nbytes: int, stream=None) -> None:
        """Device-to-device copy on the copy engines; dst may be a peer-mapped address."""
        self._check(self._lib.maize_copy_async(self._h, dst_ptr, src_ptr, nbytes, _stream_handle(stream)))

    def chain_forward(self, wait_flag_ptr, first_value: int, dst_ptr: int, src_ptr: int, total_bytes: int,
                      chunk_bytes: int, dst_flag_ptr: int, stream=None) -> None:
        """Enqueue (wait for chunk i, copy it to the next rank, publish i) for every chunk of a step in one call."""
        self._check(self._lib.maize_chain_forward(self._h, wait_flag_ptr, first_value & 0xFFFFFFFF, dst_ptr, src_ptr,
                                                  total_bytes, chunk_bytes, dst_flag_ptr, _stream_handle(stream)))

    def flags_wait(self, flags_ptr: int, count: int, value: int, stream=None) -> None:
        self._check(self._lib.maize_flags_wait(self._h, flags_ptr, count, value & 0xFFFFFFFF, _stream_handle(stream)))

    def flag_store(self, flag_ptr: int, value: int, stream=None) -> None:
        self._check(self._lib.maize_flag_store(self._h, flag_ptr, value & 0xFFFFFFFF, _stream_handle(stream)))

    def gemm_kn(self, a, b, out=None, stream=None):
        """``out = a @ b`` for bf16 CUDA tensors with b given K x N (N contiguous), the layout the reference's
        demo walks; rows may be strided."""
        import torch
        for name, t in (("a", a), ("b", b)):
            if t.dim() != 2 or t.dtype != torch.bfloat16 or not t.is_cuda or (t.shape[1] > 1 and t.stride(1) != 1):
                raise MaizeError(_ffi.INVALID_ARG, f"{name}: expected a 2-D bfloat16 CUDA tensor with unit column stride")
        m, k = a.shape
        kb, n = b.shape
        if k != kb:
            raise MaizeError(_ffi.INVALID_ARG, "a.shape[1] != b.shape[0] (b is stored K x N)")
        if out is None:
            out = torch.empty((m, n), dtype=torch.bfloat16, device=a.device)
        elif out.shape != (m, n) or out.dtype != torch.bfloat16 or not out.is_cuda or (n > 1 and out.stride(1) != 1):
            raise MaizeError(_ffi.INVALID_ARG, "out: expected an M x N bfloat16 CUDA tensor with unit column stride")
        lda = a.stride(0) if m > 1 else max(k, 8)
        ldb = b.stride(0) if k > 1 else max(n, 8)
        ldc = out.stride(0) if m > 1 else max(n, 1)
        self._check(self._lib.maize_gemm_bf16_kn_ld(self._h, a.data_ptr(), lda, b.data_ptr(), ldb, out.data_ptr(), ldc,
                                                    m, n, k, _stream_handle(stream)))
        return out

    # ------------------------------------------- products grouped by expert --
    # Small calls are bound by the host: what every call asks of its tensors is asked once and in line, and _own is only
    # there for those that fail it (or have a dimension of one with an odd stride).
    def _own(self, name: str, t, dims: int, dtype) -> None:
        """What every operand of the calls below is checked for: kind, device, unit stride along the rows."""
        if (t.dtype is not dtype or t.dim() != dims or t.get_device() != self.device
                or (t.shape[-1] > 1 and t.stride(-1) != 1)):
            raise MaizeError(_ffi.INVALID_ARG, f"{name}: expected a {dims}-D {dtype} tensor with unit column stride on "
                                               f"cuda:{self.device}")

    @staticmethod
    def _too_large(*sizes):
        """The entry points take 32-bit sizes; what passes 31 bits would arrive there cut off."""
        return MaizeError(_ffi.UNSUPPORTED, f"sizes {' x '.join(map(str, sizes))}: one is beyond the kernels' range")

    def _result(self, out, shape, dtype, stream):
        """The tensor a call writes: ``out`` if it is given and fits, else a new one, allocated for the
        stream the call runs on."""
        if out is not None:
            self._own("out", out, len(shape), dtype)
            if out.shape != shape:
                raise MaizeError(_ffi.INVALID_ARG, f"out: expected {' x '.join(map(str, shape))}")
            return out
        if stream is None:
            if _empty is not None and 0 not in shape and _current_device() == self.device:
                last = shape[-1]
                return _empty(shape, (last, 1) if len(shape) == 2 else (shape[1] * last, last, 1), dtype)
            return _torch.empty(*shape, dtype=dtype, device=_devices[self.device])
        if isinstance(stream, int):
            stream = _torch.cuda.ExternalStream(stream, device=self.device)
        with _torch.cuda.stream(stream):
            return _torch.empty(*shape, dtype=dtype, device=_devices[self.device])

    def _stream(self, stream) -> int:
        """Handle of the stream a call runs on: the given one, or the current stream of the context's device."""
        if stream is None:
            return _raw_stream(self.device)
        return stream if isinstance(stream, int) else stream.cuda_stream

    def _offsets(self, offsets, groups: int) -> None:
        if (offsets.dtype is not _torch.int32 or offsets.dim() != 1 or offsets.numel() != groups + 1
                or offsets.get_device() != self.device or not offsets.is_contiguous()):
            raise MaizeError(_ffi.INVALID_ARG, f"offsets: expected {groups + 1} contiguous int32 values on cuda:{self.device}")

    def _grouped(self, entry, a, b, offsets, out, stream, kn: bool):
        bf16, device = (_torch or _types()).bfloat16, self.device
        sa, sb = a.stride(), b.stride()
        if not (a.dtype is bf16 and b.dtype is bf16 and len(sa) == 2 and len(sb) == 3 and sa[1] == 1 and sb[2] == 1
                and a.get_device() == device and b.get_device() == device):
            self._own("a", a, 2, bf16)
            self._own("b", b, 3, bf16)
        rows, k = a.shape
        groups, b_rows, b_cols = b.shape
        n, kb = (b_cols, b_rows) if kn else (b_rows, b_cols)
        if k != kb:
            raise MaizeError(_ffi.INVALID_ARG, f"a has {k} columns, the matrices of b a K of {kb}")
        if (rows | n | k | groups) >> 31:
            raise self._too_large(rows, n, k, groups)
        self._offsets(offsets, groups)
        out = self._result(out, (rows, n), bf16, stream)
        # the stride of a dimension of one is not used and may be anything
        st = entry(self._ctx, a.data_ptr(), sa[0] if rows > 1 else -(-k // 8) * 8, b.data_ptr(),
                   sb[1] if b_rows > 1 else -(-b_cols // 8) * 8, sb[0], out.data_ptr(), out.stride(0) if rows > 1 else n,
                   offsets.data_ptr(), groups, rows, n, k, self._stream(stream))
        if st:
            self._check(st)
        return out

    def grouped_gemm(self, a, b, offsets, out=None, stream=None):
        """``out[r] = a[r] @ b[g].T`` for the rows ``offsets[g] <= r < offsets[g + 1]`` of every group g: a is rows x K,
        b is groups x N x K (one weight matrix per expert), offsets int32 on the device, ascending, groups + 1 of them.
        Rows outside all groups are left as they were.  Groups may be empty; their sizes are never read on the host."""
        return self._grouped(self._calls.maize_grouped_gemm_bf16, a, b, offsets, out, stream, False)

    def grouped_gemm_kn(self, a, b, offsets, out=None, stream=None):
        """``out[r] = a[r] @ b[g]`` with b given groups x K x N.  With ``a`` the gradient of ``grouped_gemm``'s result and
        the same b this is the gradient of its input."""
        return self._grouped(self._calls.maize_grouped_gemm_bf16_kn, a, b, offsets, out, stream, True)

    def grouped_gemm_wgrad(self, a, dc, offsets, out=None, stream=None):
        """``out[g] = dc[rows of g].T @ a[rows of g]``: the gradient of ``grouped_gemm``'s b (groups x N x K) from its
        input ``a`` (rows x K) and the gradient ``dc`` (rows x N) of its result.  A group without rows gets zeros."""
        bf16, device = (_torch or _types()).bfloat16, self.device
        sa, sd = a.stride(), dc.stride()
        if not (a.dtype is bf16 and dc.dtype is bf16 and len(sa) == 2 and len(sd) == 2 and sa[1] == 1 and sd[1] == 1
                and a.get_device() == device and dc.get_device() == device):
            self._own("a", a, 2, bf16)
            self._own("dc", dc, 2, bf16)
        rows, k = a.shape
        rows_dc, n = dc.shape
        if rows_dc != rows:
            raise MaizeError(_ffi.INVALID_ARG, f"a has {rows} rows, dc {rows_dc}")
        if (rows | n | k) >> 31:
            raise self._too_large(rows, n, k)
        groups = offsets.numel() - 1
        if groups < 0:
            raise MaizeError(_ffi.INVALID_ARG, "offsets: expected groups + 1 int32 values")
        self._offsets(offsets, groups)
        out = self._result(out, (groups, n, k), bf16, stream)
        so = out.stride()
        st = self._calls.maize_grouped_gemm_bf16_wgrad(
            self._ctx, a.data_ptr(), sa[0] if rows > 1 else -(-k // 8) * 8, dc.data_ptr(),
            sd[0] if rows > 1 else -(-n // 8) * 8, out.data_ptr(), so[1] if n > 1 else k, so[0], offsets.data_ptr(), groups, rows,
            n, k, self._stream(stream))
        if st:
            self._check(st)
        return out

    # ------------------------------------------------------ 8-bit products --
    def quantize_e4m3(self, x, block_rows: int = 1, out=None, scales=None, stream=None):
        """bf16 rows x cols -> (e4m3 tensor of the same shape, fp32 scales), with a power-of-two scale for each 1 x 128
        (``block_rows`` = 1: activations) or 128 x 128 block (``block_rows`` = 128: weights): ``x ~ q * scale``."""
        torch = _torch or _types()
        sx = x.stride()
        if not (x.dtype is torch.bfloat16 and len(sx) == 2 and sx[1] == 1 and x.get_device() == self.device):
            self._own("x", x, 2, torch.bfloat16)
        rows, cols = x.shape
        if block_rows != 1 and block_rows != 128:
            raise MaizeError(_ffi.INVALID_ARG, "block_rows must be 1 or 128")
        if (rows | cols) >> 31:
            raise self._too_large(rows, cols)
        down, across = -(-rows // block_rows), -(-cols // 128)
        out = self._result(out, (rows, cols), torch.float8_e4m3fn, stream)
        scales = self._result(scales, (down, across), torch.float32, stream)
        st = self._calls.maize_quantize_e4m3(self._ctx, x.data_ptr(), sx[0] if rows > 1 else cols, rows, cols, block_rows,
                                             out.data_ptr(), out.stride(0) if rows > 1 else cols, scales.data_ptr(),
                                             scales.stride(0) if down > 1 else across, self._stream(stream))
        if st:
            self._check(st)
        return out, scales

    def gemm_e4m3(self, a, a_scales, b, b_scales, out=None, stream=None):
        """``out = (a * a_scales) @ (b * b_scales).T`` in bf16 for e4m3 a (M x K) with a scale for each 1 x 128 block
        (M x ceil(K/128), fp32) and e4m3 b (N x K) with one for each 128 x 128 block (ceil(N/128) x ceil(K/128))."""
        torch = _torch or _types()
        f8, f32, device = torch.float8_e4m3fn, torch.float32, self.device
        sa, sb, ssa, ssb = a.stride(), b.stride(), a_scales.stride(), b_scales.stride()
        if not (a.dtype is f8 and b.dtype is f8 and a_scales.dtype is f32 and b_scales.dtype is f32
                and len(sa) == 2 and len(sb) == 2 and len(ssa) == 2 and len(ssb) == 2
                and sa[1] == 1 and sb[1] == 1 and ssa[1] == 1 and ssb[1] == 1 and a.get_device() == device
                and b.get_device() == device and a_scales.get_device() == device and b_scales.get_device() == device):
            for name, t, dtype in (("a", a, f8), ("b", b, f8), ("a_scales", a_scales, f32), ("b_scales", b_scales, f32)):
                self._own(name, t, 2, dtype)
        m, k = a.shape
        n, kb = b.shape
        if k != kb:
            raise MaizeError(_ffi.INVALID_ARG, "a.shape[1] != b.shape[1] (b is stored N x K)")
        if (m | n | k) >> 31:
            raise self._too_large(m, n, k)
        blocks, down = -(-k // 128), -(-n // 128)
        if a_scales.shape != (m, blocks) or b_scales.shape != (down, blocks):
            raise MaizeError(_ffi.INVALID_ARG, f"scales: expected {m} x {blocks} for a, {down} x {blocks} for b")
        out = self._result(out, (m, n), torch.bfloat16, stream)
        st = self._calls.maize_gemm_e4m3(self._ctx, a.data_ptr(), sa[0] if m > 1 else k, a_scales.data_ptr(),
                                         ssa[0] if m > 1 else blocks, b.data_ptr(), sb[0] if n > 1 else k, b_scales.data_ptr(),
                                         ssb[0] if down > 1 else blocks, out.data_ptr(), out.stride(0) if m > 1 else n, m, n, k,
                                         self._stream(stream))
        if st:
            self._check(st)
        return out

    def debug_wait_expires(self, budget_ns: int, stream=None) -> None:
        self._check(self._lib.maize_debug_wait_expires(self._h, int(budget_ns), _stream_handle(stream)))


_default_ctx = {}


def default_context(device: Optional[int] = None) -> Context:
    """The cached Context of a device, which the module's functions use: for one host thread at a time, like any Context."""
    import torch
    if device is None:
        device = torch.cuda.current_device()
    ctx = _default_ctx.get(device)
    if ctx is None:
        ctx = _default_ctx[device] = Context(device)
    return ctx


def gemm(a, b, out=None, stream=None):
    """``a @ b.T`` on the B200 kernels (module-level convenience over a cached Context)."""
    return default_context(a.device.index).gemm(a, b, out=out, stream=stream)


def _context_of(t) -> Context:
    device = t.get_device()
    if device < 0:
        raise MaizeError(_ffi.INVALID_ARG, "expected CUDA tensors")
    return _default_ctx.get(device) or default_context(device)


def grouped_gemm(a, b, offsets, out=None, stream=None):
    """``Context.grouped_gemm`` over a cached Context of a's device."""
    return _context_of(a).grouped_gemm(a, b, offsets, out, stream)


def grouped_gemm_kn(a, b, offsets, out=None, stream=None):
    """``Context.grouped_gemm_kn`` over a cached Context of a's device."""
    return _context_of(a).grouped_gemm_kn(a, b, offsets, out, stream)


def grouped_gemm_wgrad(a, dc, offsets, out=None, stream=None):
    """``Context.grouped_gemm_wgrad`` over a cached Context of a's device."""
    return _context_of(a).grouped_gemm_wgrad(a, dc, offsets, out, stream)


def quantize_e4m3(x, block_rows: int = 1, out=None, scales=None, stream=None):
    """``Context.quantize_e4m3`` over a cached Context of x's device."""
    return _context_of(x).quantize_e4m3(x, block_rows, out, scales, stream)


def gemm_e4m3(a, a_scales, b, b_scales, out=None, stream=None):
    """``Context.gemm_e4m3`` over a cached Context of a's device."""
    return _context_of(a).gemm_e4m3(a, a_scales, b, b_scales, out, stream)


def gemm_skinny_static(a, b, out, stream=None, device_status=None):
    """``out = a @ b.T`` for M <= 32 through the entry point that allocates nothing.

    For callers that may not allocate device memory at this point (so ``out`` must be passed in): the
    kernel's scratch is a fixed array inside the library (8 MiB per GPU).  Shapes beyond what that array
    can serve raise ``MaizeError(UNSUPPORTED)`` with the sizes in the message.  Calls that could overlap
    on the GPU share the array and must be ordered by the caller.  ``device_status``: optional int32[4]
    CUDA tensor that receives a timeout code.
    """
    import torch
    lib = _ffi.load()
    err = ctypes.create_string_buffer(256)
    # the C entry assumes dense rows (lda = ldb = K, ldc = N) on the current device: check before handing out pointers
    cur = torch.cuda.current_device()
    for name, t in (("a", a), ("b", b), ("out", out)):
        if (t.dim() != 2 or t.dtype != torch.bfloat16 or not t.is_cuda or t.device.index != cur
                or (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) != t.shape[1])):
            raise MaizeError(_ffi.INVALID_ARG, f"{name}: expected a dense 2-D bfloat16 tensor on the current CUDA device")
    if device_status is not None and (device_status.dtype != torch.int32 or device_status.numel() < 4
                                      or not device_status.is_cuda or not device_status.is_contiguous()):
        raise MaizeError(_ffi.INVALID_ARG, "device_status: expected a contiguous int32 CUDA tensor of at least 4 elements")
    m, k = a.shape
    n, kb = b.shape
    st = lib.maize_gemm_bf16_skinny_static(a.data_ptr(), m, k, b.data_ptr(), n, kb, out.data_ptr(), out.shape[0],
                                           out.shape[1], _stream_handle(stream),
                                           device_status.data_ptr() if device_status is not None else None,
                                           err, len(err))
    if st != _ffi.OK:
        raise MaizeError(st, err.value.decode())
    return out
