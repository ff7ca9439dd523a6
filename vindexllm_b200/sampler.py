"""Host-side mirror of VindexLLM's sampler interface over the C ABI.

``TVdxSampler`` keeps the reference's method names and meaning (src/VindexLLM.Sampler.pas:
DefaultConfig :100-109, SetConfig :132-150, GetConfig :152-155, Process :265-528,
AddToHistory :530-539, ResetHistory :541-549) for a batch of rows, each with its own
PRNG and history ring. ``SamplerContext.sample`` is the stateless batched call
(vdxs_sample_ex). torch only supplies device memory and streams; all sampling runs in
libvdxsampler.so, and a missing library raises instead of falling back.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import abi
from ._lib import load, check, VdxsError
from .abi import VdxsConfig, default_config

__all__ = ["SamplerContext", "TVdxSampler", "ShardComm", "DeviceDecodeState", "Q4Weights", "I8Weights", "BeamSearch",
           "BeamState", "VdxsError", "default_config", "shard_range", "broadcast_unique_id"]


def _stream_ptr(stream):
    import torch
    if stream is None:
        stream = torch.cuda.current_stream()
    return C.c_void_p(int(stream.cuda_stream))


def _dtype_code(t) -> int:
    import torch
    if t.dtype == torch.float32:
        return abi.DTYPE_F32
    if t.dtype == torch.bfloat16:
        return abi.DTYPE_BF16
    raise TypeError(f"logits must be float32 or bfloat16, got {t.dtype}")


def _dptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _ptr(t):
    """Address of a tensor, as ctypes takes it for a pointer argument (0 is NULL)."""
    return 0 if t is None else t.data_ptr()


_HIDDEN_CODES: dict = {}


def _hidden_code(t, what: str) -> int:
    """VDXS_DTYPE_* of a hidden state or norm weight."""
    if not _HIDDEN_CODES:
        import torch
        _HIDDEN_CODES.update({torch.float32: abi.DTYPE_F32, torch.bfloat16: abi.DTYPE_BF16,
                              torch.float16: abi.DTYPE_F16})
    code = _HIDDEN_CODES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


_raw_stream = None


def _stream_on(device: int, stream) -> int:
    """The stream of a call on `device`: the given one, or the device's current one."""
    global _raw_stream
    if stream is not None:
        return stream.cuda_stream
    if _raw_stream is None:
        import torch
        # The handle of current_stream(device) without the object around it (1.3 us a call).
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                              lambda d: torch.cuda.current_stream(d).cuda_stream)
    return _raw_stream(device)


def _output(like, dtype, stream, *shape):
    """An output on the device of `like`. With a stream of the caller's it is allocated under that
    one, so that its memory is reused in that stream's order."""
    if stream is not None:
        import torch
        with torch.cuda.stream(stream):
            return like.new_empty(shape, dtype=dtype)
    # Sizes one by one and no keyword: 1.3 us a call instead of 2.2.
    return like.new_empty(*shape) if like.dtype is dtype else like.new_empty(*shape, dtype=dtype)


def _need(t, what: str, device: int, dtype, shape):
    """Checks a contiguous tensor's device, type and shape (dtype or shape None: any)."""
    if t.get_device() != device:
        raise ValueError(f"{what} must be a tensor on cuda:{device}, got {t.device}")
    if dtype is not None and t.dtype is not dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{what} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")


def _matrix(t, what: str, device: int, dtype, shape) -> int:
    """Checks a matrix with contiguous rows (dtype None: any); returns the elements between its
    rows (a lone row's stride says nothing)."""
    if t.get_device() != device:
        raise ValueError(f"{what} must be a tensor on cuda:{device}, got {t.device}")
    if dtype is not None and t.dtype is not dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{what} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    stride = t.stride()
    if len(stride) != 2 or (stride[1] != 1 and shape[1] > 1):
        raise ValueError(f"{what} must be a matrix with contiguous rows")
    return stride[0] if shape[0] > 1 else max(stride[0], shape[1])


class SamplerContext:
    """One vdxs_context: a device plus its lazily grown workspace."""

    def __init__(self, device: int = 0, tie_mode: int = abi.TIES_FAITHFUL):
        self.lib = load()
        h = C.c_void_p()
        check(self.lib.vdxs_create(device, C.byref(h)))
        self._h = h
        self.device = device
        self.set_tie_mode(tie_mode)

    @property
    def handle(self):
        return self._h

    def close(self):
        if getattr(self, "_h", None):
            self.lib.vdxs_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def set_tie_mode(self, mode: int):
        check(self.lib.vdxs_set_tie_mode(self._h, mode), self._h)

    def device_status(self, stream=None):
        """vdxs_device_status: waits for the stream, raises VdxsError if a kernel of an
        earlier call reported a timeout or a failed internal check."""
        check(self.lib.vdxs_device_status(self._h, _stream_ptr(stream)), self._h)

    def set_stage_events(self, ev_begin=None, ev_end=None):
        """Records two torch.cuda.Event objects around the dominant pass of every later
        call (None, None stops). The events are created here if torch has not yet."""
        if ev_begin is None or ev_end is None:
            check(self.lib.vdxs_set_stage_events(self._h, None, None), self._h)
            return
        for ev in (ev_begin, ev_end):
            if not ev.cuda_event:
                ev.record()
        check(self.lib.vdxs_set_stage_events(self._h, C.c_void_p(ev_begin.cuda_event),
                                             C.c_void_p(ev_end.cuda_event)), self._h)

    def launch_count(self) -> int:
        """Kernels the library has launched for this context."""
        n = C.c_int64()
        check(self.lib.vdxs_get_launch_count(self._h, C.byref(n)), self._h)
        return n.value

    def sample(self, cfg: VdxsConfig, logits, uniforms=None, history=None, history_count=None,
               vocab: int | None = None, out_k: int = 0, want_flags: bool = False, stream=None,
               tokens=None):
        """Stateless batched sampling on device tensors. Returns tokens, or
        (tokens, flags, idx, prob) when diagnostics are requested."""
        import torch
        assert logits.is_cuda and logits.dim() == 2 and logits.stride(1) == 1
        B, _ = logits.shape
        V = logits.shape[1] if vocab is None else vocab
        dev = logits.device
        if tokens is None:
            tokens = torch.empty(B, dtype=torch.int32, device=dev)
        flags = torch.empty(B, dtype=torch.int32, device=dev) if (want_flags or out_k) else None
        oi = torch.empty(B, out_k, dtype=torch.int32, device=dev) if out_k else None
        op = torch.empty(B, out_k, dtype=torch.float32, device=dev) if out_k else None
        hs = history.shape[1] if history is not None else 1
        rc = self.lib.vdxs_sample_ex(self._h, C.byref(cfg), _dptr(logits), _dtype_code(logits), B, V,
                                     logits.stride(0), _dptr(history), hs, _dptr(history_count),
                                     _dptr(uniforms), _dptr(tokens), _dptr(flags), _dptr(oi), _dptr(op),
                                     out_k, _stream_ptr(stream))
        check(rc, self._h)
        if flags is None:
            return tokens
        return tokens, flags, oi, op

    def rms_norm_i8(self, x, weight, eps: float = 1e-6, residual=None, out_hidden=None, q=None, scale=None,
                    stream=None):
        """vdxs_rms_norm_i8: (q, scale, hidden) of the rows of ``x`` [rows, dim]; hidden is
        x + residual (None without a residual and without ``out_hidden``). ``out_hidden`` may be
        ``x`` or ``residual`` for an update in place. A ``q`` made here has rows padded to a
        multiple of 16 bytes, as ``I8Weights.unembed`` takes it."""
        import torch
        dev, dtype, shape = self.device, x.dtype, x.shape
        code, wcode = _hidden_code(x, "x"), _hidden_code(weight, "weight")
        pitch = _matrix(x, "x", dev, None, shape)
        rows, dim = shape
        _need(weight, "weight", dev, None, (dim,))
        rp = hp = 0
        if residual is not None:
            rp = _matrix(residual, "residual", dev, dtype, shape)
            if out_hidden is None:
                out_hidden, hp = _output(x, dtype, stream, rows, dim), dim
        if out_hidden is not None and not hp:
            hp = _matrix(out_hidden, "out_hidden", dev, dtype, shape)
        if q is None:
            qp = -(-dim // 16) * 16
            q = _output(x, torch.int8, stream, rows, qp)
            if qp != dim:
                q = q[:, :dim]
        else:
            qp = _matrix(q, "q", dev, torch.int8, shape)
        if scale is None:
            scale = _output(weight, torch.float32, stream, rows)
        else:
            _need(scale, "scale", dev, torch.float32, (rows,))
        rc = self.lib.vdxs_rms_norm_i8(self._h, x.data_ptr(), pitch, _ptr(residual), rp, code, weight.data_ptr(), wcode,
                                       rows, dim, eps, _ptr(out_hidden), hp, q.data_ptr(), qp, scale.data_ptr(),
                                       _stream_on(dev, stream))
        if rc:
            check(rc, self._h)
        return q, scale, out_hidden

    def sample_host(self, cfg: VdxsConfig, logits: np.ndarray, uniforms=None, history=None,
                    history_count=None, vocab: int | None = None, stream=None, out=None):
        """Host-buffer call (vdxs_sample_host): numpy (or pinned torch CPU) inputs, host tokens."""
        lg = logits
        if hasattr(lg, "numpy"):
            lg = lg.numpy()
        if lg.dtype == np.float32:
            dt = abi.DTYPE_F32
        elif lg.dtype in (np.uint16, np.int16):
            dt = abi.DTYPE_BF16
        else:
            raise TypeError("host logits must be float32 or bf16 bits (uint16)")
        B, S = lg.shape
        V = S if vocab is None else vocab
        out = np.empty(B, np.int32) if out is None else out

        def p(a):
            if a is None:
                return None
            if hasattr(a, "numpy"):
                a = a.numpy()
            return C.c_void_p(a.ctypes.data)
        hs = history.shape[1] if history is not None else 1
        rc = self.lib.vdxs_sample_host(self._h, C.byref(cfg), p(lg), dt, B, V, S, p(history), hs,
                                       p(history_count), p(uniforms), C.c_void_p(out.ctypes.data),
                                       _stream_ptr(stream) if stream is not None else None)
        check(rc, self._h)
        return out


class TVdxSampler:
    """TVdxSampler (Sampler.pas:37-91) for ``batch`` independent rows."""

    DefaultConfig = staticmethod(default_config)

    def __init__(self, ctx: SamplerContext, batch: int = 1):
        self.ctx = ctx
        self.lib = ctx.lib
        self.batch = batch
        h = C.c_void_p()
        check(self.lib.vdxs_sampler_create(ctx.handle, batch, C.byref(h)), ctx.handle)
        self._h = h

    def close(self):
        if getattr(self, "_h", None):
            self.lib.vdxs_sampler_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def SetConfig(self, cfg: VdxsConfig):
        check(self.lib.vdxs_sampler_set_config(self._h, C.byref(cfg)), self.ctx.handle)

    def GetConfig(self) -> VdxsConfig:
        c = VdxsConfig()
        check(self.lib.vdxs_sampler_get_config(self._h, C.byref(c)), self.ctx.handle)
        return c

    def AddToHistory(self, token: int, row: int = 0):
        check(self.lib.vdxs_sampler_add_to_history(self._h, row, int(token)), self.ctx.handle)

    def AddToHistoryBatch(self, tokens):
        t = np.ascontiguousarray(tokens, dtype=np.int32)
        check(self.lib.vdxs_sampler_add_to_history_batch(self._h, C.c_void_p(t.ctypes.data)), self.ctx.handle)

    def ResetHistory(self, row: int = -1):
        check(self.lib.vdxs_sampler_reset_history(self._h, row), self.ctx.handle)

    def Process(self, logits, vocab: int | None = None, stream=None):
        """Process for every row. ``logits``: a CUDA tensor [batch, stride] (fp32/bf16), or a
        host float32 array [batch, stride] (the reference's PSingle calling shape).
        Returns an int32 numpy array of token ids (a Python int when batch == 1)."""
        out = np.empty(self.batch, np.int32)
        if isinstance(logits, np.ndarray):
            assert logits.dtype == np.float32 and logits.ndim in (1, 2)
            lg = np.ascontiguousarray(logits.reshape(self.batch, -1))
            V = lg.shape[1] if vocab is None else vocab
            check(self.lib.vdxs_sampler_process_host(self._h, C.c_void_p(lg.ctypes.data), V, lg.shape[1],
                                                     C.c_void_p(out.ctypes.data)), self.ctx.handle)
        else:
            lg = logits.reshape(self.batch, -1) if logits.dim() == 1 else logits
            V = lg.shape[1] if vocab is None else vocab
            check(self.lib.vdxs_sampler_process(self._h, _dptr(lg), _dtype_code(lg), V, lg.stride(0),
                                                C.c_void_p(out.ctypes.data), _stream_ptr(stream)),
                  self.ctx.handle)
        return int(out[0]) if self.batch == 1 else out

    def NextFloat(self, row: int = 0) -> float:
        f = C.c_float()
        check(self.lib.vdxs_sampler_next_float(self._h, row, C.byref(f)), self.ctx.handle)
        return f.value

    def GetPrngState(self, row: int = 0):
        st = (C.c_uint64 * 4)()
        check(self.lib.vdxs_sampler_get_prng_state(self._h, row, st), self.ctx.handle)
        return list(st)

    def SetPrngState(self, state, row: int = 0):
        check(self.lib.vdxs_sampler_set_prng_state(self._h, row, (C.c_uint64 * 4)(*state)), self.ctx.handle)

    def GetHistory(self, row: int = 0):
        cap = max(1, self.GetConfig().repeat_window)
        buf = (C.c_int32 * cap)()
        cnt, pos = C.c_int32(), C.c_int32()
        check(self.lib.vdxs_sampler_get_history(self._h, row, buf, cap, C.byref(cnt), C.byref(pos)),
              self.ctx.handle)
        return list(buf[: cnt.value]), cnt.value, pos.value


class DeviceDecodeState:
    """Row PRNGs and history rings kept on the device (vdxs_device_uniforms,
    vdxs_device_history_push, vdxs_decode_step), so a decode loop samples without a host
    round trip per token. The reference keeps both inside TVdxSampler on the host
    (Sampler.pas:157-248 PRNG, :530-549 ring); ``prng_states`` takes their 4-word states,
    e.g. from ``TVdxSampler.GetPrngState``."""

    def __init__(self, batch: int, window: int, device: int = 0, prng_states=None):
        import torch
        dev = torch.device("cuda", device)
        self.lib = load()
        self.batch, self.window = batch, window
        self.prng = torch.zeros((batch, 4), dtype=torch.int64, device=dev)  # uint64 bit patterns
        if prng_states is not None:
            st = np.ascontiguousarray(np.asarray(prng_states, dtype=np.uint64).reshape(batch, 4)).view(np.int64)
            self.prng.copy_(torch.from_numpy(st))
        self.uniforms = torch.zeros(batch, dtype=torch.float32, device=dev)
        self.hist = torch.zeros((batch, max(window, 1)), dtype=torch.int32, device=dev)
        self.pos = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.count = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.stopped = torch.zeros(batch, dtype=torch.int32, device=dev)

    def next_uniforms(self, stream=None):
        """One NextFloat per row (Sampler.pas:243-248); returns the device tensor."""
        check(self.lib.vdxs_device_uniforms(_dptr(self.prng), self.batch, _dptr(self.uniforms), _stream_ptr(stream)))
        return self.uniforms

    def push(self, tokens, stop_ids=None, stream=None):
        """AddToHistory (Sampler.pas:530-539) of device tokens[batch]; flags stop tokens."""
        n_stop = 0 if stop_ids is None else int(stop_ids.numel())
        check(self.lib.vdxs_device_history_push(_dptr(self.hist), _dptr(self.pos), _dptr(self.count), self.window,
                                                _dptr(tokens), self.batch, _dptr(stop_ids), n_stop,
                                                _dptr(self.stopped), _stream_ptr(stream)))

    def step(self, ctx: "SamplerContext", cfg: VdxsConfig, logits, stop_ids=None, tokens=None, stream=None):
        """One device-resident decode step (vdxs_decode_step); returns the device tokens."""
        import torch
        assert logits.is_cuda and logits.dim() == 2 and logits.stride(1) == 1
        B, V = logits.shape
        assert B == self.batch and cfg.repeat_window == self.window
        if tokens is None:
            tokens = torch.empty(B, dtype=torch.int32, device=logits.device)
        n_stop = 0 if stop_ids is None else int(stop_ids.numel())
        check(self.lib.vdxs_decode_step(ctx._h, C.byref(cfg), _dptr(logits), _dtype_code(logits), B, V,
                                        logits.stride(0), _dptr(self.prng), _dptr(self.uniforms), _dptr(self.hist),
                                        _dptr(self.pos), _dptr(self.count), _dptr(stop_ids), n_stop,
                                        _dptr(self.stopped), _dptr(tokens), _stream_ptr(stream)), ctx._h)
        return tokens


def shard_range(vocab: int, world: int, rank: int) -> tuple[int, int]:
    """Contiguous vocab shard [lo, hi) of `rank`: the first vocab % world ranks hold one
    extra token, so every id has exactly one owner and shards are in rank order."""
    if world < 1 or not 0 <= rank < world:
        raise ValueError(f"rank {rank} of world {world}")
    q, r = divmod(vocab, world)
    lo = rank * q + min(rank, r)
    return lo, lo + q + (1 if rank < r else 0)


def broadcast_unique_id(rank: int, src: int = 0) -> bytes:
    """NCCL unique id made on `src` and shared through the caller's torch.distributed
    process group (any backend): what each rank passes to ShardComm."""
    import torch.distributed as dist
    obj = [ShardComm.unique_id() if rank == src else None]
    dist.broadcast_object_list(obj, src=src)
    return obj[0]


class ShardComm:
    """An NCCL communicator owned by the library (vdxs_comm)."""

    def __init__(self, ctx: SamplerContext, nranks: int, rank: int, unique_id: bytes, timeout_ms: int = 60000):
        """Creates the communicator (non-blocking NCCL init under `timeout_ms`: a rank that
        never joins raises VdxsError with VDXS_E_TIMEOUT instead of hanging)."""
        self.ctx = ctx
        self.lib = ctx.lib
        assert len(unique_id) == 128
        buf = (C.c_uint8 * 128).from_buffer_copy(unique_id)
        h = C.c_void_p()
        check(self.lib.vdxs_comm_create_ex(ctx.handle, nranks, rank, buf, int(timeout_ms), C.byref(h)), ctx.handle)
        self._h = h
        self.nranks = nranks
        self.rank = rank

    @staticmethod
    def unique_id() -> bytes:
        lib = load()
        buf = (C.c_uint8 * 128)()
        check(lib.vdxs_comm_unique_id(buf))
        return bytes(buf)

    def close(self):
        if getattr(self, "_h", None):
            self.lib.vdxs_comm_destroy(self._h)
            self._h = None

    def abort(self):
        """vdxs_comm_abort: for a caller that learned on the host that a peer left."""
        check(self.lib.vdxs_comm_abort(self._h), self.ctx.handle)

    def status(self):
        """vdxs_comm_status: raises VdxsError after an asynchronous NCCL error or an abort."""
        check(self.lib.vdxs_comm_status(self._h), self.ctx.handle)

    def wait(self, stream=None, timeout_ms: int = 0):
        """vdxs_comm_wait: bounded wait for the stream; aborts the communicator on failure."""
        check(self.lib.vdxs_comm_wait(self._h, _stream_ptr(stream), int(timeout_ms)), self.ctx.handle)

    def sample(self, cfg: VdxsConfig, logits_shard, vocab_offset: int, vocab_total: int, uniforms=None,
               history=None, history_count=None, want_flags: bool = False, stream=None, tokens=None):
        import torch
        B, V = logits_shard.shape
        if tokens is None:
            tokens = torch.empty(B, dtype=torch.int32, device=logits_shard.device)
        flags = torch.empty(B, dtype=torch.int32, device=logits_shard.device) if want_flags else None
        hs = history.shape[1] if history is not None else 1
        rc = self.lib.vdxs_sample_sharded(self.ctx.handle, self._h, C.byref(cfg), _dptr(logits_shard),
                                          _dtype_code(logits_shard), B, V, logits_shard.stride(0),
                                          vocab_offset, vocab_total, _dptr(history), hs, _dptr(history_count),
                                          _dptr(uniforms), _dptr(tokens), _dptr(flags), _stream_ptr(stream))
        check(rc, self.ctx.handle)
        return (tokens, flags) if want_flags else tokens


class Q4Weights:
    """A Q4_0 unembedding matrix prepared on a context's device (vdxs_q4_0_prepare):
    TVdxModel.UnembedToLogits (src/VindexLLM.Model.pas:1258-1271) with the matvec of
    shaders/matvec_q4_0.comp, in front of the sampler."""

    def __init__(self, ctx: SamplerContext, q4_0, in_dim: int, out_dim: int, stream=None):
        """``q4_0``: a uint8 CUDA tensor holding [out_dim, in_dim / 32 * 18] Q4_0 blocks."""
        assert q4_0.is_cuda and q4_0.is_contiguous() and q4_0.numel() == out_dim * (in_dim // 32) * 18
        self.ctx = ctx
        self.lib = ctx.lib
        self.in_dim, self.out_dim = in_dim, out_dim
        h = C.c_void_p()
        check(self.lib.vdxs_q4_0_prepare(ctx.handle, _dptr(q4_0), in_dim, out_dim, _stream_ptr(stream),
                                         C.byref(h)), ctx.handle)
        self._h = h

    def close(self):
        if getattr(self, "_h", None):
            self.lib.vdxs_q4_0_release(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def unembed(self, hidden, logits=None, stream=None):
        """logits [batch, out_dim] float32 = hidden [batch, in_dim] x weights^T."""
        import torch
        assert hidden.is_cuda and hidden.dtype == torch.float32 and hidden.is_contiguous()
        hidden = hidden.reshape(-1, self.in_dim)
        if logits is None:
            logits = torch.empty(hidden.shape[0], self.out_dim, dtype=torch.float32, device=hidden.device)
        check(self.lib.vdxs_unembed_q4_0(self.ctx.handle, self._h, _dptr(hidden), hidden.shape[0], _dptr(logits),
                                         _stream_ptr(stream)), self.ctx.handle)
        return logits

    def sample(self, cfg: VdxsConfig, hidden, uniforms=None, history=None, history_count=None, tokens=None,
               stream=None):
        """vdxs_sample_unembed_q4_0: unembedding and sampling in one call; returns tokens."""
        import torch
        assert hidden.is_cuda and hidden.dtype == torch.float32 and hidden.is_contiguous()
        hidden = hidden.reshape(-1, self.in_dim)
        B = hidden.shape[0]
        if tokens is None:
            tokens = torch.empty(B, dtype=torch.int32, device=hidden.device)
        hs = history.shape[1] if history is not None else 1
        check(self.lib.vdxs_sample_unembed_q4_0(self.ctx.handle, C.byref(cfg), self._h, _dptr(hidden), B,
                                                _dptr(history), hs, _dptr(history_count), _dptr(uniforms),
                                                _dptr(tokens), _stream_ptr(stream)), self.ctx.handle)
        return tokens


class I8Weights:
    """An unembedding matrix in 8-bit integers with a scale for each vocabulary entry
    (vdxs_i8_prepare): the final norm, the product on the integer tensor cores and the
    sampler for every batch size. Stands beside Q4Weights, whose matvec keeps the reference's
    order of sums and serves small batches."""

    def __init__(self, ctx: SamplerContext, weight, scales=None, stream=None):
        """``weight`` [out_dim, in_dim]: int8 with ``scales`` [out_dim] float32, or float32,
        bfloat16 or float16, quantised here row by row."""
        import torch
        formats = {torch.float32: abi.WEIGHTS_F32, torch.bfloat16: abi.WEIGHTS_BF16, torch.float16: abi.WEIGHTS_F16,
                   torch.int8: abi.WEIGHTS_I8}
        if weight.dtype not in formats:
            raise TypeError(f"weight must be int8, float32, bfloat16 or float16, got {weight.dtype}")
        pitch = _matrix(weight, "weight", ctx.device, None, weight.shape)
        out_dim, in_dim = weight.shape
        if (weight.dtype == torch.int8) != (scales is not None):
            raise ValueError("scales go with int8 weights, and with those alone")
        if scales is not None:
            _need(scales, "scales", ctx.device, torch.float32, (out_dim,))
        self._prepare(ctx, weight, formats[weight.dtype], scales, pitch, in_dim, out_dim, stream)

    @classmethod
    def from_q4_0(cls, ctx: SamplerContext, q4_0, in_dim: int, out_dim: int, stream=None) -> "I8Weights":
        """From the reference's Q4_0 blocks (the uint8 tensor that Q4Weights takes)."""
        import torch
        _need(q4_0, "q4_0", ctx.device, torch.uint8, None)
        if q4_0.numel() != out_dim * (in_dim // 32) * 18:
            raise ValueError(f"{q4_0.numel()} bytes are not {out_dim} x {in_dim} in Q4_0 blocks")
        w = cls.__new__(cls)
        w._prepare(ctx, q4_0, abi.WEIGHTS_Q4_0, None, in_dim, in_dim, out_dim, stream)
        return w

    def _prepare(self, ctx, weight, fmt, scales, stride, in_dim, out_dim, stream):
        self.ctx, self.lib = ctx, ctx.lib
        self.in_dim, self.out_dim = in_dim, out_dim
        h = C.c_void_p()
        check(self.lib.vdxs_i8_prepare(ctx.handle, _ptr(weight), fmt, _ptr(scales), stride, in_dim, out_dim,
                                       _stream_on(ctx.device, stream), C.byref(h)), ctx.handle)
        self._h = h

    def close(self):
        if getattr(self, "_h", None):
            self.lib.vdxs_i8_release(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def unembed(self, q, scale, logits=None, dtype=None, stream=None):
        """logits [batch, out_dim] (float32 or bfloat16) of 8-bit rows ``q`` [batch, in_dim] with
        ``scale`` [batch], as SamplerContext.rms_norm_i8 returns them."""
        import torch
        dev, batch, n = self.ctx.device, q.shape[0], self.out_dim
        qp = _matrix(q, "q", dev, torch.int8, (batch, self.in_dim))
        if batch == 1:
            qp = -(-self.in_dim // 16) * 16
        _need(scale, "scale", dev, torch.float32, (batch,))
        if logits is None:
            logits, pitch = _output(scale, dtype or torch.float32, stream, batch, n), n
        else:
            pitch = _matrix(logits, "logits", dev, dtype, (batch, n))
        rc = self.lib.vdxs_unembed_i8(self.ctx._h, self._h, q.data_ptr(), qp, scale.data_ptr(), batch, logits.data_ptr(),
                                      _dtype_code(logits), pitch, _stream_on(dev, stream))
        if rc:
            check(rc, self.ctx._h)
        return logits

    def sample(self, cfg: VdxsConfig, x, norm_weight, eps: float = 1e-6, residual=None, out_hidden=None, uniforms=None,
               history=None, history_count=None, tokens=None, stream=None):
        """vdxs_sample_unembed_i8: norm, unembedding and sampling in one call; returns tokens."""
        import torch
        dev, batch = self.ctx.device, x.shape[0]
        shape = (batch, self.in_dim)
        code, wcode = _hidden_code(x, "x"), _hidden_code(norm_weight, "norm_weight")
        pitch = _matrix(x, "x", dev, None, shape)
        rp = 0 if residual is None else _matrix(residual, "residual", dev, x.dtype, shape)
        hp = 0 if out_hidden is None else _matrix(out_hidden, "out_hidden", dev, x.dtype, shape)
        _need(norm_weight, "norm_weight", dev, None, (self.in_dim,))
        if tokens is None:
            tokens = _output(x, torch.int32, stream, batch)
        for t, what, dtype in ((uniforms, "uniforms", torch.float32), (history_count, "history_count", torch.int32),
                               (tokens, "tokens", torch.int32)):
            if t is not None:
                _need(t, what, dev, dtype, (batch,))
        hs = 1
        if history is not None:
            hs = history.shape[1]
            _need(history, "history", dev, torch.int32, (batch, hs))
        check(self.lib.vdxs_sample_unembed_i8(self.ctx._h, C.byref(cfg), self._h, x.data_ptr(), pitch, _ptr(residual), rp,
                                              code, norm_weight.data_ptr(), wcode, eps, _ptr(out_hidden), hp, batch,
                                              _ptr(history), hs, _ptr(history_count), _ptr(uniforms), tokens.data_ptr(),
                                              _stream_on(dev, stream)), self.ctx._h)
        return tokens


class BeamState:
    """Device state of a search's batch * beams rows (vdxs_beam_rows): cumulative scores,
    lengths, finished flags and, with window > 0, the penalty rings. A new state is that of
    a search at its start: beam 0 of each prompt has score 0, the others -infinity."""

    def __init__(self, batch: int, beams: int, window: int = 0, device=None, scores=None, lengths=None, finished=None,
                 hist=None, pos=None, count=None):
        import torch
        if device is None:
            device = scores.device if scores is not None else torch.cuda.current_device()
        device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        rows = batch * beams
        self.batch, self.beams, self.window = batch, beams, window

        def own(t, dtype, *shape):
            if t is None:
                return torch.zeros(shape, dtype=dtype, device=device)
            _need(t, "state", device.index, dtype, shape)
            return t

        if scores is None:
            scores = torch.full((batch, beams), -float("inf"), dtype=torch.float32, device=device)
            scores[:, 0] = 0.0
            scores = scores.view(-1)
        self.scores = own(scores, torch.float32, rows)
        self.lengths = own(lengths, torch.int32, rows)
        self.finished = own(finished, torch.int32, rows)
        self.hist = own(hist, torch.int32, rows, window) if window else None
        self.pos = own(pos, torch.int32, rows) if window else None
        self.count = own(count, torch.int32, rows) if window else None

    def rows(self) -> abi.VdxsBeamRows:
        if not self.window:
            return abi.VdxsBeamRows(self.scores.data_ptr(), self.lengths.data_ptr(), self.finished.data_ptr())
        return abi.VdxsBeamRows(self.scores.data_ptr(), self.lengths.data_ptr(), self.finished.data_ptr(),
                                self.hist.data_ptr(), self.pos.data_ptr(), self.count.data_ptr())


def _cache_pieces(t, what: str, most: int | None = None):
    """(row stride, segment stride, segment bytes, segments) of a tensor [rows, ...] whose rows are
    one contiguous piece, or equal pieces (of at most `most` bytes) at one distance."""
    size, shape, stride = t.element_size(), t.shape, t.stride()
    inner = count = 1
    d = len(shape) - 1
    while d > 0 and (shape[d] == 1 or (stride[d] == inner and (most is None or inner * size < most))):
        inner *= shape[d]
        d -= 1
    step = inner
    while d > 0:
        n, s = shape[d], stride[d]
        d -= 1
        if n == 1:
            continue
        if count == 1:
            step = s
        elif s != step * count:
            raise ValueError(f"{what}: the rows of strides {stride} are not equal pieces at one distance")
        count *= n
    row = stride[0] if shape[0] > 1 else step * count
    return row * size, step * size, inner * size, count


class BeamSearch:
    """A beam search of ``batch`` prompts with ``beams`` beams each over ``vocab`` tokens
    (vdxs_beam): the selection over beams and vocabulary, with the reordering of the rows.
    The reference decodes one sequence and has no counterpart."""

    def __init__(self, ctx: SamplerContext, batch: int, beams: int, vocab: int):
        self.ctx, self.lib = ctx, ctx.lib
        self.batch, self.beams, self.vocab = batch, beams, vocab
        h = C.c_void_p()
        check(self.lib.vdxs_beam_create(ctx.handle, batch, beams, vocab, C.byref(h)), ctx.handle)
        self._h = h

    def close(self):
        if getattr(self, "_h", None):
            self.lib.vdxs_beam_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _handle(self):
        """The search's handle, which points to its context's."""
        if not self.ctx._h:
            raise VdxsError(abi.E_INVALID_ARG, "the search's context is closed")
        return self._h

    def _caches(self, caches):
        """A cache is a tensor [rows, ...] (in place) or a pair (source, target) of them; a view
        of the filled part moves that part alone."""
        n = len(caches)
        if not n:
            return None, 0
        out = (abi.VdxsBeamCache * n)()
        dev, rows = self.ctx.device, self.batch * self.beams
        for i, c in enumerate(caches):
            src, dst = c if isinstance(c, (tuple, list)) else (c, c)
            for t in (src, dst):
                if t.get_device() != dev:
                    raise ValueError(f"cache {i} must be on cuda:{dev}, got {t.device}")
                if t.dim() < 1 or t.shape[0] != rows:
                    raise ValueError(f"cache {i} must have {rows} rows, got shape {tuple(t.shape)}")
            if src is not dst and (src.shape != dst.shape or src.dtype != dst.dtype):
                raise ValueError(f"cache {i}: source and target differ in shape or type")
            if src.numel() == 0:
                continue  # a zeroed entry has no bytes to move
            a = b = _cache_pieces(src, f"cache {i}")
            if src is not dst:
                b = _cache_pieces(dst, f"cache {i}")
            if a[2] != b[2]:  # the smaller pieces of the two
                a, b = (_cache_pieces(t, f"cache {i}", min(a[2], b[2])) for t in (src, dst))
            if a[2:] != b[2:]:
                raise ValueError(f"cache {i}: source and target are laid out in different pieces")
            out[i] = abi.VdxsBeamCache(src.data_ptr(), dst.data_ptr(), a[0], a[1], b[0], b[1], a[2], a[3])
        return out, n

    def step(self, state: BeamState, logits, out: BeamState | None = None, stop_ids=None, pad_token: int = 0,
             repeat_penalty: float = 1.0, length_alpha: float = 0.0, caches=(), tokens=None, parents=None, stream=None):
        """One step (vdxs_beam_step): (tokens, parents) as int32 [batch, beams]. ``out`` receives the
        rows after it (``state`` itself, in place, when None). A cache that layers share is listed
        once."""
        import torch
        h = self._handle()
        dev, batch, beams, i32 = self.ctx.device, self.batch, self.beams, torch.int32
        shape = (batch, beams)
        pitch = _matrix(logits, "logits", dev, None, (batch * beams, self.vocab))
        self._check_state(state, state.window)
        a = b = state.rows()
        if out is not None and out is not state:
            self._check_state(out, state.window)
            b = out.rows()
        n_stop = 0
        if stop_ids is not None:
            _need(stop_ids, "stop_ids", dev, i32, None)
            n_stop = stop_ids.numel()
        if tokens is None:
            tokens = _output(state.finished, i32, stream, batch, beams)
        else:
            _need(tokens, "tokens", dev, i32, shape)
        if parents is None:
            parents = _output(state.finished, i32, stream, batch, beams)
        else:
            _need(parents, "parents", dev, i32, shape)
        cfg = abi.VdxsBeamConfig(length_alpha, repeat_penalty, state.window, pad_token, 0)
        moved, n = self._caches(caches) if caches else (None, 0)
        rc = self.lib.vdxs_beam_step(h, C.byref(cfg), logits.data_ptr(), _dtype_code(logits), pitch, C.byref(a),
                                     C.byref(b), _ptr(stop_ids), n_stop, moved, n, tokens.data_ptr(), parents.data_ptr(),
                                     _stream_on(dev, stream))
        if rc:
            check(rc, self.ctx._h)
        return tokens, parents

    def _check_state(self, s: BeamState, window: int):
        if s.batch != self.batch or s.beams != self.beams or s.window != window:
            raise ValueError(f"a state of {s.batch} x {s.beams}, window {s.window}, for a search of {self.batch} x "
                             f"{self.beams}, window {window}")
        if s.scores.get_device() != self.ctx.device:
            raise ValueError(f"the state is on {s.scores.device}, the search on cuda:{self.ctx.device}")

    def reorder(self, parents, caches, stream=None):
        """Moves caches by a step's parents (vdxs_beam_reorder)."""
        import torch
        h = self._handle()
        _need(parents, "parents", self.ctx.device, torch.int32, (self.batch, self.beams))
        moved, n = self._caches(caches)
        check(self.lib.vdxs_beam_reorder(h, _ptr(parents), moved, n, _stream_on(self.ctx.device, stream)),
              self.ctx._h)
