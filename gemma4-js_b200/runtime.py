"""Host-side mirror of the reference's GPU operator API over the g4w4 C ABI.

The reference model graph (custom-webgpu/gemma4-webgpu.js) talks to its runtime
through `GPUOps` (custom-webgpu/gpu-runtime.js:1295-1378), `GPUW4Linear.load`
(:1385-1392), `reader.pleRowsToGpu(device, ids)` (:905, :993, :1050) and `KVCache`
(gemma4-webgpu.js:122-137).  This module exposes the same operators with the same
argument meaning and the same errors (raised as G4Error), over libg4w4.so.
Device buffers are torch CUDA tensors; like the reference, each operator returns
a newly allocated output.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import _lib
from ._lib import G4_BF16, G4_F32, G4Error, G4Rows, G4Sampling, G4Tree, call

_DT = {torch.float32: G4_F32, torch.bfloat16: G4_BF16}


def _ptr(t: torch.Tensor) -> C.c_void_p:
    return C.c_void_p(t.data_ptr())


def _host_or_device(a) -> tuple[C.c_void_p, int, object]:
    """(pointer, on_device, keepalive) for a numpy array or a contiguous torch tensor."""
    if isinstance(a, torch.Tensor):
        a = a.contiguous()
        return C.c_void_p(a.data_ptr()), int(a.is_cuda), a
    a = np.ascontiguousarray(a)
    return C.c_void_p(a.ctypes.data), 0, a


def _need(ctx: "Context", name: str, what: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple | None = None) -> int:
    """The device pointer of a contiguous tensor argument of the context's device, type and shape."""
    if t.dtype is not dtype or t.device != ctx.torch_device or not t.is_contiguous() or (
            shape is not None and t.shape != shape):
        raise G4Error(-1, f"{name}: {what} must be a contiguous {dtype} tensor"
                          f"{'' if shape is None else f' of shape {shape}'} on {ctx.torch_device}, got {t.dtype} "
                          f"{tuple(t.shape)} with strides {tuple(t.stride())} on {t.device}")
    return t.data_ptr()


class Context:
    """One g4_ctx per GPU (the reference's WebGPU device + queue)."""

    def __init__(self, device: int = 0, stream: torch.cuda.Stream | None = None):
        _lib.load()
        self.device = device
        self.torch_device = torch.device("cuda", device)
        s = stream if stream is not None else torch.cuda.current_stream(self.torch_device)
        self._stream, self._raw_stream = s, s.cuda_stream
        h = C.c_void_p()
        call("g4_ctx_create", device, C.c_void_p(s.cuda_stream), C.byref(h))
        self.handle = h

    def set_stream(self, stream: torch.cuda.Stream) -> None:
        self._stream, self._raw_stream = stream, stream.cuda_stream
        call("g4_ctx_set_stream", self.handle, C.c_void_p(stream.cuda_stream))

    def set_pdl(self, enable: bool) -> None:
        """Programmatic dependent launch for this context's kernels (g4_ctx_set_pdl)."""
        call("g4_ctx_set_pdl", self.handle, int(bool(enable)))

    @property
    def stream(self) -> torch.cuda.Stream:
        return self._stream

    def sync(self) -> None:
        call("g4_stream_sync", self.handle)

    def empty(self, shape, dtype: torch.dtype, *used: torch.Tensor | None) -> torch.Tensor:
        """An output tensor of a call on this context's stream.  When that is not torch's current
        stream, the output comes from the context stream's own memory (a block that torch still
        uses elsewhere cannot be handed out early), and the call's inputs (`used`) are not reused
        before the context stream is done with them."""
        if torch._C._cuda_getCurrentRawStream(self.device) == self._raw_stream:
            return torch.empty(shape, dtype=dtype, device=self.torch_device)
        self.use(*used)
        with torch.cuda.stream(self._stream):
            return torch.empty(shape, dtype=dtype, device=self.torch_device)

    def use(self, *tensors: torch.Tensor | None) -> None:
        """The context stream is going to read or write these: when it is not torch's current stream, their
        memory is not handed out again before it is done with them."""
        if torch._C._cuda_getCurrentRawStream(self.device) == self._raw_stream:
            return
        for t in tensors:
            if t is not None:
                t.record_stream(self._stream)

    def empty_like(self, t: torch.Tensor, dtype: torch.dtype, *used: torch.Tensor | None) -> torch.Tensor:
        """empty() in the shape of a contiguous t (which torch makes in half the time)."""
        if torch._C._cuda_getCurrentRawStream(self.device) == self._raw_stream:
            return torch.empty_like(t, dtype=dtype)
        return self.empty(t.shape, dtype, t, *used)

    def fill(self, t: torch.Tensor, value) -> None:
        """t.fill_(value) on the context's stream."""
        with torch.cuda.stream(self._stream):
            t.fill_(value)

    def check_device(self) -> int:
        """Raises G4Error if a kernel raised the device error word since the last check."""
        flags = C.c_uint32(0)
        st = _lib.load().g4_ctx_check_device(self.handle, C.byref(flags))
        _lib.check(st)
        return flags.value

    def close(self) -> None:
        if getattr(self, "handle", None):
            _lib.load().g4_ctx_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class W4Linear:
    """GPUW4Linear (gpu-runtime.js:1380-1394): packed int32 [N, K/8] + bf16 scales [N, K/group]."""

    def __init__(self, ctx: Context, packed, scales, group_size: int = 32, name: str = ""):
        self.ctx = ctx
        self.name = name
        out_dim = int(packed.shape[0])
        in_dim = int(packed.shape[1]) * 8
        groups = int(scales.shape[1])
        if groups == 0 or in_dim % groups:
            raise G4Error(-1, f"{name}: scale shape {tuple(scales.shape)} does not divide K={in_dim}")
        group_size = in_dim // groups  # gpu-runtime.js:1388 derives it from the shapes
        if isinstance(scales, torch.Tensor) and scales.dtype == torch.bfloat16:
            scales = scales.view(torch.int16)
        pp, pd, keep1 = _host_or_device(packed)
        sp, sd, keep2 = _host_or_device(scales)
        if pd != sd:
            raise G4Error(-1, "packed and scales must both be on the host or both on the device")
        h = C.c_void_p()
        call("g4_linear_create", ctx.handle, pp, sp, in_dim, out_dim, group_size, pd, C.byref(h))
        self.handle = h
        self.in_dim, self.out_dim, self.group_size, self.groups = in_dim, out_dim, group_size, groups

    def dequant(self, row_start: int = 0, row_count: int | None = None, dtype=torch.float32) -> torch.Tensor:
        rc = self.out_dim - row_start if row_count is None else row_count
        out = torch.empty((rc, self.in_dim), dtype=dtype, device=self.ctx.torch_device)
        call("g4_linear_dequant", self.ctx.handle, self.handle, row_start, rc, _ptr(out), _DT[dtype])
        return out

    def close(self):
        if getattr(self, "handle", None):
            _lib.load().g4_linear_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class PleW4Table:
    """Device-resident PLE W4 table; rows_to_gpu mirrors reader.pleRowsToGpu(device, ids)."""

    def __init__(self, ctx: Context, packed, scales, vocab: int | None = None, width: int = 8960, group: int = 32):
        self.ctx = ctx
        if packed is None:
            assert vocab is not None
            h = C.c_void_p()
            call("g4_ple_table_create", ctx.handle, None, None, vocab, width, group, 0, C.byref(h))
        else:
            vocab = int(packed.shape[0])
            width = int(packed.shape[1]) * 2
            if isinstance(scales, torch.Tensor) and scales.dtype == torch.bfloat16:
                scales = scales.view(torch.int16)
            pp, pd, k1 = _host_or_device(packed)
            sp, sd, k2 = _host_or_device(scales)
            h = C.c_void_p()
            call("g4_ple_table_create", ctx.handle, pp, sp, vocab, width, group, pd, C.byref(h))
        self.handle = h
        self.vocab, self.width, self.group = vocab, width, group

    def upload_rows(self, row_start: int, packed, scales) -> None:
        pp, pd, k1 = _host_or_device(packed)
        sp, sd, k2 = _host_or_device(scales)
        call("g4_ple_table_upload_rows", self.ctx.handle, self.handle, row_start, int(packed.shape[0]), pp, sp, pd)
        if pd:
            self.ctx.sync()

    def rows_to_gpu(self, ids, dtype=torch.float32, out: torch.Tensor | None = None) -> torch.Tensor:
        """[T, width] dequantised rows (f32 like the reference, or bf16)."""
        if isinstance(ids, torch.Tensor) and ids.is_cuda:
            ids_t = ids.to(torch.int32).contiguous()
            T, ptr, on_dev, keep = ids_t.numel(), _ptr(ids_t), 1, ids_t
        else:
            arr = np.ascontiguousarray(np.asarray(ids, dtype=np.int64))
            if arr.size and (arr.min() < -(2**31) or arr.max() >= 2**31):
                raise G4Error(-6, f"PLE token id out of range: {int(arr.max())}")
            keep = arr.astype(np.int32)
            T, ptr, on_dev = keep.size, C.c_void_p(keep.ctypes.data), 0
        if out is None:
            out = torch.empty((T, self.width), dtype=dtype, device=self.ctx.torch_device)
        call("g4_ple_gather", self.ctx.handle, self.handle, ptr, T, on_dev, _ptr(out), _DT[out.dtype])
        return out

    def close(self):
        if getattr(self, "handle", None):
            _lib.load().g4_ple_table_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class KVCache:
    """KVCache (gemma4-webgpu.js:122-137) with bf16 storage.

    ring > 0: a sliding-window cache of `nseq` sequences that keeps each sequence's last
    `ring` positions (g4_kv_create_ring); max_seq stays the position limit.  `rows` is the
    storage height and `seq_rows` the row stride per sequence."""

    def __init__(self, ctx: Context, head_dim: int, max_seq: int, ring: int = 0, nseq: int = 1):
        self.ctx = ctx
        h = C.c_void_p()
        if ring:
            call("g4_kv_create_ring", ctx.handle, head_dim, max_seq, ring, nseq, C.byref(h))
        else:
            call("g4_kv_create", ctx.handle, head_dim, max_seq, C.byref(h))
        self.handle = h
        self.head_dim, self.max_seq = head_dim, max_seq
        r, sr, n = C.c_int(0), C.c_int(0), C.c_int(0)
        call("g4_kv_layout", h, C.byref(r), C.byref(sr), C.byref(n))
        self.ring, self.seq_rows, self.nseq = r.value, sr.value, n.value
        self.rows = self.seq_rows * self.nseq if self.ring else max_seq

    def slot(self, pos: int) -> int:
        """Storage row of position pos (of sequence 0)."""
        return pos % self.ring if self.ring else pos

    @property
    def length(self) -> int:
        n = C.c_int(0)
        call("g4_kv_info", self.handle, C.byref(n), None, None)
        return n.value

    def append(self, k: torch.Tensor, v: torch.Tensor, rows: int, start_pos: int) -> None:
        k = k.contiguous()
        v = v.contiguous()
        if k.dtype != v.dtype or k.dtype not in _DT:
            raise G4Error(-1, "KV append wants f32 or bf16 k and v of one dtype")
        call("g4_kv_append", self.ctx.handle, self.handle, _ptr(k), _ptr(v), rows, start_pos, _DT[k.dtype])

    def reset(self) -> None:
        call("g4_kv_reset", self.handle)

    def storage(self) -> tuple[torch.Tensor, torch.Tensor]:
        """The bf16 K and V storage [rows, head_dim] itself, as tensors that share its memory
        and keep the cache alive.  The library reads and writes it on the context's stream."""
        kp, vp = C.c_void_p(), C.c_void_p()
        call("g4_kv_buffers", self.handle, C.byref(kp), C.byref(vp))
        return tuple(torch.as_tensor(_Storage(self, p.value), device=self.ctx.torch_device).view(torch.bfloat16)
                     for p in (kp, vp))

    def tensors(self) -> tuple[torch.Tensor, torch.Tensor]:
        """Copies of the bf16 K and V storage [rows, head_dim] (for tests)."""
        kp, vp = C.c_void_p(), C.c_void_p()
        call("g4_kv_buffers", self.handle, C.byref(kp), C.byref(vp))
        n = self.rows * self.head_dim
        return _wrap_device(kp.value, n, self.ctx).view(self.rows, self.head_dim), \
            _wrap_device(vp.value, n, self.ctx).view(self.rows, self.head_dim)

    def close(self):
        if getattr(self, "handle", None):
            _lib.load().g4_kv_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class _Storage:
    """A cache's K or V storage for torch.as_tensor (no copy; the tensor keeps this object)."""

    def __init__(self, cache: KVCache, ptr: int):
        self.cache = cache
        self.__cuda_array_interface__ = {"shape": (cache.rows, cache.head_dim), "typestr": "<i2", "strides": None,
                                         "data": (ptr, False), "version": 2}


def _cache_table(caches) -> C.Array:
    return (C.c_void_p * len(caches))(*[c.handle for c in caches])


def _seq_stride(caches, seq_stride: int | None) -> int:
    """Rows per sequence of the linear caches (a ring cache has its own): all of them by default."""
    return seq_stride or min((c.rows for c in caches if not c.ring), default=1)


def kv_compact(ctx: Context, caches, seq_pos: torch.Tensor, path: torch.Tensor, accepted: torch.Tensor,
               seq_stride: int | None = None, seq_base: int = 0) -> None:
    """Moves the accepted rows of drafted trees together behind the cached ones, in every cache of
    the list at once (g4_kv_compact): path int32 [nseq, nodes] and accepted int32 [nseq] as
    GPUOps.treeAccept returns them, seq_pos the int32 positions before the drafted tokens."""
    nseq, nodes = path.shape
    pp = _need(ctx, "kv_compact", "path", path, torch.int32)
    ap = _need(ctx, "kv_compact", "accepted", accepted, torch.int32, (nseq,))
    sp = _need(ctx, "kv_compact", "seq_pos", seq_pos, torch.int32)
    if seq_base < 0 or seq_base + nseq > seq_pos.numel():
        raise G4Error(-6, f"kv_compact: sequences {seq_base}..{seq_base + nseq} of {seq_pos.numel()} positions")
    ctx.use(seq_pos, path, accepted)
    call("g4_kv_compact", ctx.handle, _cache_table(caches), len(caches), _seq_stride(caches, seq_stride), sp, seq_base,
         nseq, nodes, pp, ap)


def kv_fork(ctx: Context, caches, seq_pos: torch.Tensor, src, dst, seq_stride: int | None = None) -> None:
    """Copies the cached rows and the position of sequence src[i] to sequence dst[i], in every cache
    of the list at once (g4_kv_fork); src and dst are sequences of ints on the host."""
    src, dst = [int(i) for i in src], [int(i) for i in dst]
    if len(src) != len(dst):
        raise G4Error(-1, f"kv_fork: {len(src)} sources, {len(dst)} destinations")
    sp = _need(ctx, "kv_fork", "seq_pos", seq_pos, torch.int32)
    n = len(src)
    if any(not 0 <= i < seq_pos.numel() for i in (*src, *dst)):
        raise G4Error(-6, f"kv_fork: sequences {src} -> {dst} of {seq_pos.numel()} positions")
    ctx.use(seq_pos)
    call("g4_kv_fork", ctx.handle, _cache_table(caches), len(caches), _seq_stride(caches, seq_stride), sp,
         (C.c_int32 * n)(*src), (C.c_int32 * n)(*dst), n)


def _wrap_device(ptr: int, n: int, ctx: Context) -> torch.Tensor:
    """Copies n bf16 values from a library-owned device pointer into a new tensor."""
    out = torch.empty(n, dtype=torch.bfloat16, device=ctx.torch_device)
    ctx.sync()
    cudart = C.CDLL("libcudart.so.12")
    cudart.cudaMemcpy.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
    res = cudart.cudaMemcpy(C.c_void_p(out.data_ptr()), C.c_void_p(ptr), n * 2, 3)  # device to device
    if int(res) != 0:
        raise G4Error(-3, f"cudaMemcpy failed ({res})")
    return out


class GPUOps:
    """GPUOps (gpu-runtime.js:1295-1378) over libg4w4, method for method.

    Every operator takes and returns the reference's f32 buffers (a new output per call,
    like `emptyF32`); w4 and attention also take bf16 activations (the W4A16 kernels'
    own input type), returning bf16 unless asked otherwise."""

    def __init__(self, ctx: Context):
        self.ctx = ctx

    def _f32(self, n: int) -> torch.Tensor:
        return torch.empty(n, dtype=torch.float32, device=self.ctx.torch_device)

    @staticmethod
    def _need_f32(name: str, *ts: torch.Tensor) -> None:
        for t in ts:
            if t.dtype != torch.float32:
                raise G4Error(-1, f"{name}: f32 buffers expected, got {t.dtype}")

    def w4(self, linear: W4Linear, x: torch.Tensor, rows: int, out_dtype=None, impl: int = 0,
           out: torch.Tensor | None = None) -> torch.Tensor:
        """GPUOps.w4(encoder, linear, x, rows): y[rows, outDim] = x . dequant(W)^T.  f32 x (the
        reference's buffers) gives f32 y through g4_linear_w4a16_f32; bf16 x runs the kernels
        directly (bf16 out unless out_dtype / out say f32)."""
        x = x.contiguous()
        if x.numel() != rows * linear.in_dim:
            raise G4Error(-1, f"{linear.name}: x has {x.numel()} values, expected {rows}x{linear.in_dim}")
        if x.dtype == torch.float32:
            if impl != 0 or (out_dtype not in (None, torch.float32)):
                raise G4Error(-1, f"{linear.name}: f32 x gives f32 y through the automatic kernel choice")
            if out is None:
                out = torch.empty((rows, linear.out_dim), dtype=torch.float32, device=self.ctx.torch_device)
            call("g4_linear_w4a16_f32", self.ctx.handle, linear.handle, _ptr(x), rows, _ptr(out))
            return out
        if x.dtype != torch.bfloat16:
            raise G4Error(-1, f"{linear.name}: x must be f32 or bf16, got {x.dtype}")
        if out is None:
            out = torch.empty((rows, linear.out_dim), dtype=out_dtype or torch.bfloat16, device=self.ctx.torch_device)
        call("g4_linear_w4a16_impl", self.ctx.handle, linear.handle, _ptr(x), rows, _ptr(out), _DT[out.dtype], impl)
        return out

    def rms(self, x: torch.Tensor, rows: int, width: int, scale: torch.Tensor | None = None) -> torch.Tensor:
        """GPUOps.rms(encoder, x, rows, width, scale) (RMS_SHADER, eps 1e-6)."""
        self._need_f32("rms", x, *([scale] if scale is not None else []))
        y = self._f32(rows * width)
        call("g4_rms", self.ctx.handle, _ptr(x), _ptr(scale) if scale is not None else None, rows, width,
             C.c_float(1e-6), _ptr(y), G4_F32)
        return y

    def addScale(self, a: torch.Tensor, b: torch.Tensor, n: int, scale: float = 1.0) -> torch.Tensor:  # noqa: N802
        """GPUOps.addScale(encoder, a, b, n, scale)."""
        self._need_f32("addScale", a, b)
        y = self._f32(n)
        call("g4_add_scale", self.ctx.handle, _ptr(a), _ptr(b), n, C.c_float(scale), _ptr(y))
        return y

    def scale(self, a: torch.Tensor, n: int, s: float) -> torch.Tensor:
        """GPUOps.scale(encoder, a, n, s)."""
        self._need_f32("scale", a)
        y = self._f32(n)
        call("g4_scale", self.ctx.handle, _ptr(a), n, C.c_float(s), _ptr(y))
        return y

    def geluMul(self, gate: torch.Tensor, up: torch.Tensor, n: int) -> torch.Tensor:  # noqa: N802
        """GPUOps.geluMul(encoder, gate, up, n)."""
        self._need_f32("geluMul", gate, up)
        y = self._f32(n)
        call("g4_gelu_mul_f32", self.ctx.handle, _ptr(gate), _ptr(up), n, _ptr(y))
        return y

    def geluPle(self, gate: torch.Tensor, ple: torch.Tensor, rows: int, layer: int,  # noqa: N802
                layers: int = 35, dim: int = 256) -> torch.Tensor:
        """GPUOps.geluPle(encoder, gate, ple, rows, layer): ple is [rows, 35, 256]."""
        self._need_f32("geluPle", gate, ple)
        y = self._f32(rows * dim)
        call("g4_gelu_ple_f32", self.ctx.handle, _ptr(gate), _ptr(ple), rows, layer, layers, dim, _ptr(y))
        return y

    def normRope(self, x: torch.Tensor, rows: int, heads: int, hd: int, pos0: int, scale: torch.Tensor,  # noqa: N802
                 ropeProp: float, base: float) -> torch.Tensor:  # noqa: N803
        """GPUOps.normRope(encoder, x, rows, heads, hd, pos0, scale, ropeProp, base)."""
        self._need_f32("normRope", x, scale)
        y = self._f32(rows * heads * hd)
        call("g4_norm_rope", self.ctx.handle, _ptr(x), rows, heads, hd, pos0, _ptr(scale), int(ropeProp * hd / 2),
             C.c_float(base), C.c_float(1e-6), _ptr(y))
        return y

    def attention(self, q: torch.Tensor, cache: KVCache, qrows: int, heads: int, hd: int, keylen: int,
                  qpos0: int, sliding: bool, window: int, out: torch.Tensor | None = None) -> torch.Tensor:
        """GPUOps.attention(encoder, q, kcache, vcache, qrows, heads, hd, keylen, qpos0, sliding, window):
        the cache object stands for the reference's kcache/vcache pair.  f32 q (the reference's
        buffers) gives an f32 result through g4_attention_f32; bf16 q gives bf16."""
        q = q.contiguous()
        if q.dtype == torch.float32:
            if out is None:
                out = torch.empty((qrows, heads, hd), dtype=torch.float32, device=self.ctx.torch_device)
            call("g4_attention_f32", self.ctx.handle, _ptr(q), cache.handle, qrows, heads, hd, keylen, qpos0,
                 int(bool(sliding)), window, _ptr(out))
            return out
        if q.dtype != torch.bfloat16:
            raise G4Error(-1, f"attention: q must be f32 or bf16, got {q.dtype}")
        if out is None:
            out = torch.empty((qrows, heads, hd), dtype=torch.bfloat16, device=self.ctx.torch_device)
        call("g4_attention", self.ctx.handle, _ptr(q), cache.handle, qrows, heads, hd, keylen, qpos0,
             int(bool(sliding)), window, _ptr(out))
        return out

    def pleMix(self, proj: torch.Tensor, normScale: torch.Tensor, tokenPle: torch.Tensor, rows: int,  # noqa: N802,N803
               layers: int = 35, dim: int = 256) -> torch.Tensor:
        """GPUOps.pleMix(encoder, proj, normScale, tokenPle, rows): the reference scales proj
        beforehand (ops.scale by 1/sqrt(hidden)); proj here is that scaled projection."""
        self._need_f32("pleMix", proj, normScale, tokenPle)
        y = self._f32(rows * layers * dim)
        call("g4_ple_mix", self.ctx.handle, _ptr(proj), C.c_float(1.0), _ptr(normScale), _ptr(tokenPle), rows,
             layers, dim, C.c_float(1e-6), _ptr(y))
        return y


    # ---- sampling and drafted trees (no counterpart in the reference, which answers greedily) ----
    def sample(self, logits: torch.Tensor, uniform: torch.Tensor, temperature: torch.Tensor | None = None,
               top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None,
               cap: float = 0.0) -> tuple[torch.Tensor, torch.Tensor]:
        """One token per row of f32 logits [rows, vocab] (rows may be strided) from one uniform
        number per row: (ids int32 [rows], probs f32 [rows]) of g4_sample.  The settings are
        device tensors of one entry per row (f32; top_k int32), None = off."""
        if logits.dtype != torch.float32 or logits.dim() != 2 or logits.device != self.ctx.torch_device or (
                logits.shape[1] > 1 and logits.stride(1) != 1):
            raise G4Error(-1, f"sample: logits must be f32 [rows, vocab] rows on {self.ctx.torch_device}, got "
                              f"{logits.dtype} {tuple(logits.shape)} strides {logits.stride()} on {logits.device}")
        ctx, f32 = self.ctx, torch.float32
        rows, vocab = logits.shape
        ld = logits.stride(0) if rows > 1 else vocab
        shape = (rows,)
        how = G4Sampling(None if temperature is None else _need(ctx, "sample", "temperature", temperature, f32, shape),
                         None if top_k is None else _need(ctx, "sample", "top_k", top_k, torch.int32, shape),
                         None if top_p is None else _need(ctx, "sample", "top_p", top_p, f32, shape),
                         None if min_p is None else _need(ctx, "sample", "min_p", min_p, f32, shape),
                         _need(ctx, "sample", "uniform", uniform, f32, shape))
        ids = ctx.empty_like(uniform, torch.int32, logits, temperature, top_k, top_p, min_p)
        probs = ctx.empty_like(uniform, f32)
        call("g4_sample", self.ctx.handle, logits.data_ptr(), ld, rows, vocab, cap, C.byref(how), ids.data_ptr(),
             probs.data_ptr())
        return ids, probs

    def _tree(self, name: str, parents: torch.Tensor, nseq: int, nodes: int, counts: torch.Tensor | None) -> G4Tree:
        shared = parents.dim() == 1
        pp = _need(self.ctx, name, "parents", parents, torch.int32, (nodes,) if shared else (nseq, nodes))
        return G4Tree(pp, 0 if shared else nodes, nodes,
                      None if counts is None else _need(self.ctx, name, "counts", counts, torch.int32, (nseq,)))

    def attentionTree(self, q: torch.Tensor, cache: KVCache, seq_pos: torch.Tensor, parents: torch.Tensor,  # noqa: N802
                      counts: torch.Tensor | None = None, seq_stride: int | None = None, seq_base: int = 0,
                      sliding: bool = False, window: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of drafted trees (g4_attention_tree): q bf16 [nseq, nodes, heads, hd], the
        drafted rows' K/V already in the cache at seq_pos + node; parents int32 [nseq, nodes], or
        [nodes] for one tree of all sequences.  Rows behind a sequence's count keep what `out`
        held (0 in a new one)."""
        if q.dim() != 4:
            raise G4Error(-1, f"attentionTree: q must be [nseq, nodes, heads, hd], got {tuple(q.shape)}")
        nseq, nodes, heads, hd = q.shape
        qp = _need(self.ctx, "attentionTree", "q", q, torch.bfloat16)
        sp = _need(self.ctx, "attentionTree", "seq_pos", seq_pos, torch.int32)
        if seq_base < 0 or seq_base + nseq > seq_pos.numel():
            raise G4Error(-6, f"attentionTree: sequences {seq_base}..{seq_base + nseq} of {seq_pos.numel()} positions")
        tree = self._tree("attentionTree", parents, nseq, nodes, counts)
        if out is None:
            out = self.ctx.empty_like(q, torch.bfloat16, seq_pos, parents, counts)
            if counts is not None:  # rows that no node writes
                self.ctx.fill(out, 0)
            op = out.data_ptr()
        else:
            op = _need(self.ctx, "attentionTree", "out", out, torch.bfloat16, q.shape)
            self.ctx.use(q, seq_pos, parents, counts, out)
        rmap = G4Rows(sp, seq_base, nodes, 0, 0)
        call("g4_attention_tree", self.ctx.handle, qp, cache.handle, nseq * nodes, heads, hd, C.byref(rmap),
             C.byref(tree), cache.seq_rows if cache.ring else _seq_stride([cache], seq_stride), int(bool(sliding)), window,
             op)
        return out

    def treeAccept(self, parents: torch.Tensor, tokens: torch.Tensor, picks: torch.Tensor,  # noqa: N802
                   counts: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """The accepted path of each drafted tree (g4_tree_accept): tokens and picks int32
        [nseq, nodes]; returns (path [nseq, nodes], accepted [nseq], next [nseq]), int32 (next is
        -1 for a sequence without nodes)."""
        nseq, nodes = tokens.shape
        tp = _need(self.ctx, "treeAccept", "tokens", tokens, torch.int32)
        kp = _need(self.ctx, "treeAccept", "picks", picks, torch.int32, (nseq, nodes))
        tree = self._tree("treeAccept", parents, nseq, nodes, counts)
        path = self.ctx.empty_like(tokens, torch.int32, parents, picks, counts)
        accepted = self.ctx.empty(nseq, torch.int32)
        nxt = self.ctx.empty(nseq, torch.int32)
        if counts is not None:
            self.ctx.fill(nxt, -1)
        call("g4_tree_accept", self.ctx.handle, C.byref(tree), nseq, tp, kp, path.data_ptr(), accepted.data_ptr(),
             nxt.data_ptr())
        return path, accepted, nxt


def launch_count() -> int:
    return int(_lib.load().g4_kernel_launch_count())
