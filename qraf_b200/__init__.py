"""qraf_b200 — B200-native block-quantized (Q8_0 / Q4_0) matvec for QRAF.

Host-side Python mirror of the reference's operator API for this one path
(simonpierreboucher02/qraf: ``qraf::dispatch_matvec_q`` in src/nn/backend.cpp:131-199,
``dot_q8_0_f32`` / ``dot_q4_0_f32`` and ``quantize_q8_0`` / ``quantize_q4_0`` in
src/tensor/quantize.cpp), calling the sm_100a kernels of ``libqraf_cuda.so``
through its C ABI (include/qraf_cuda.h).  PyTorch is used only to hold device
memory and streams.

There is no CPU fallback: every compute entry point runs on the GPU, and
the first call into it raises ImportError if the CUDA library has not been
built.
"""
from __future__ import annotations

import ctypes as C
import os
import weakref

import numpy as np

from . import build as _build

Q8_0 = 10
Q4_0 = 20

MODE_EXACT = 0
MODE_FAST = 1
MODE_TC = 2
MODE_AUTO = 3
MODE_FLAG_OVERLAP = 0x100
MODEL_F32 = 1               # qraf_cuda_model_open_ex: upload the F32 tensors too
DECODER_KV_INT8 = 1         # qraf_cuda_decoder_open_ex: int8 KV cache (the reference's QuantizedKVCache)

OK = 0
ERR_INVALID = 1
ERR_UNSUPPORTED = 2
ERR_CUDA = 3
ERR_TIMEOUT = 4
ERR_COMM = 5
ERR_NOMEM = 6

LIB_PATH = _build.LIB


class QrafError(RuntimeError):
    """A non-zero status from the C ABI (the reference raises QrafError too, include/core/error.h)."""

    def __init__(self, code: int, msg: str):
        super().__init__(f"qraf_cuda error {code}: {msg}")
        self.code = code


class qraf_weight_t(C.Structure):
    _fields_ = [
        ("data", C.c_void_p),
        ("bytes", C.c_uint64),
        ("row_bytes", C.c_uint64),
        ("dtype", C.c_uint32),
        ("block_size", C.c_uint32),
        ("rows", C.c_uint32),
        ("cols", C.c_uint32),
        ("device", C.c_int32),
        ("owned", C.c_uint32),
    ]


class qraf_kv_t(C.Structure):
    _fields_ = [
        ("k", C.c_void_p),
        ("v", C.c_void_p),
        ("k_scale", C.c_void_p),
        ("v_scale", C.c_void_p),
        ("slot_rows", C.c_uint64),
        ("slots", C.c_uint32),
        ("rows", C.c_uint32),
        ("kv_heads", C.c_uint32),
        ("head_dim", C.c_uint32),
        ("device", C.c_int32),
    ]


def _load() -> C.CDLL:
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"{LIB_PATH} is missing: run `python -m qraf_b200.build` (nvcc, sm_100a) first")
    lib = C.CDLL(LIB_PATH)
    W, KV = C.POINTER(qraf_weight_t), C.POINTER(qraf_kv_t)
    vp, u32, u64, i32, f32p = C.c_void_p, C.c_uint32, C.c_uint64, C.c_int, C.POINTER(C.c_float)
    sig = {
        "qraf_cuda_version": (C.c_char_p, []),
        "qraf_cuda_init": (i32, [i32]),
        "qraf_cuda_shutdown": (i32, []),
        "qraf_cuda_last_error": (i32, [C.c_char_p, C.c_size_t]),
        "qraf_cuda_device_status": (i32, [i32]),
        "qraf_row_bytes": (u64, [u32, u32, u32]),
        "qraf_cuda_weight_wrap": (i32, [vp, u64, u32, u32, u32, u32, W]),
        "qraf_cuda_weight_upload": (i32, [vp, u64, u32, u32, u32, u32, W]),
        "qraf_cuda_weight_free": (i32, [W]),
        "qraf_cuda_weight_shard": (i32, [W, u32, u32, W]),
        "qraf_cuda_matvec_q": (i32, [W, vp, vp, u32, i32, vp]),
        "qraf_cuda_matvec_q_multi": (i32, [W, u32, vp, C.POINTER(vp), u32, i32, vp]),
        "qraf_cuda_matvec_q_swiglu": (i32, [W, W, vp, vp, u32, i32, vp]),
        "qraf_cuda_matvec_q_multi_ex": (i32, [W, u32, vp, vp, C.c_float, C.POINTER(vp), C.POINTER(vp), u32, i32, vp]),
        "qraf_cuda_matvec_q_swiglu_ex": (i32, [W, W, vp, vp, C.c_float, vp, u32, i32, vp]),
        "qraf_cuda_matmul_tc_noalloc": (i32, [W, vp, vp, u32, i32, vp]),
        "qraf_cuda_dot_q": (i32, [u32, vp, vp, u64, u32, vp, i32, vp]),
        "qraf_cuda_block_partials": (i32, [W, vp, vp, vp]),
        "qraf_cuda_limb_partials": (i32, [W, vp, vp, vp, vp]),
        "qraf_cuda_quantize": (i32, [u32, vp, u64, u32, vp, vp]),
        "qraf_cuda_quantize_rows": (i32, [u32, vp, u32, u32, u32, vp, vp]),
        "qraf_cuda_dequantize": (i32, [u32, vp, u64, u32, vp, vp]),
        "qraf_cuda_matvec_q_host": (i32, [vp, u64, u32, u32, u32, u32, vp, vp, u32, i32]),
        "qraf_cuda_host_cache_clear": (i32, []),
        "qraf_cuda_host_cache_add": (i32, [vp, u64, u32, u32, u32, u32]),
        "qraf_cuda_host_cache_info": (i32, [C.POINTER(u32), C.POINTER(u64)]),
        "qraf_cuda_model_open": (i32, [C.c_char_p, C.POINTER(vp)]),
        "qraf_cuda_model_weight": (i32, [vp, C.c_char_p, W]),
        "qraf_cuda_model_info": (i32, [vp, C.POINTER(u32), C.POINTER(u64), C.POINTER(i32)]),
        "qraf_cuda_model_weight_name": (C.c_char_p, [vp, u32]),
        "qraf_cuda_model_config_u32": (i32, [vp, C.c_char_p, C.POINTER(u32)]),
        "qraf_cuda_model_close": (i32, [vp]),
        "qraf_cuda_launch_count": (u64, []),
        "qraf_cuda_decoder_open": (i32, [C.c_char_p, u32, u32, C.POINTER(vp)]),
        "qraf_cuda_decoder_step": (i32, [vp, u32, vp, vp, vp, vp, i32, vp]),
        "qraf_cuda_decoder_info": (i32, [vp, C.POINTER(u32), C.POINTER(u32), C.POINTER(u32), C.POINTER(u32),
                                         C.POINTER(u32)]),
        "qraf_cuda_decoder_close": (i32, [vp]),
        "qraf_cuda_decoder_open_ex": (i32, [C.c_char_p, u32, u32, u32, C.POINTER(vp)]),
        "qraf_cuda_decoder_kv_read": (i32, [vp, u32, u32, u32, vp, vp, f32p, f32p]),
        "qraf_cuda_model_open_ex": (i32, [C.c_char_p, u32, C.POINTER(vp)]),
        "qraf_cuda_model_tensor_f32": (i32, [vp, C.c_char_p, C.POINTER(vp), C.POINTER(u64)]),
        "qraf_cuda_kv_wrap": (i32, [vp, vp, vp, vp, u32, u32, u64, u32, u32, KV]),
        "qraf_cuda_kv_store": (i32, [KV, vp, vp, u32, u64, u64, u32, vp, vp, vp, u32, vp]),
        "qraf_cuda_kv_load": (i32, [KV, vp, vp, u32, u64, u64, u32, vp, vp, vp, u32, vp]),
        "qraf_cuda_kv_attention": (i32, [KV, KV, u32, u32, vp, vp, u32, u64, u64, u32, u32, vp, vp, vp, u32, u32,
                                         C.c_float, vp, u64, vp]),
        "qraf_cuda_kv_attention_workspace": (i32, [KV, u32, u32, u32, u32, i32, u32, C.POINTER(u64)]),
        "qraf_cuda_decoder_kv": (i32, [vp, u32, KV]),
        "qraf_cuda_decoder_share_prefix": (i32, [vp, u32, u32]),
        "qraf_cuda_decoder_step_runs": (i32, [vp, u32, vp, vp, vp, vp, u32, vp, i32, vp]),
        "qraf_cuda_token_probs": (i32, [vp, u64, vp, u64, u32, u32, C.c_float, vp]),
        "qraf_cuda_verify_drafts": (i32, [vp, u64, u64, vp, u64, u64, vp, vp, vp, vp, u32, u32, u32, vp, vp, vp]),
        "qraf_fill_normal": (None, [u32, C.c_float, C.c_float, f32p, u64]),
        "qraf_cuda_comm_create": (i32, [i32, i32, u64, C.POINTER(vp)]),
        "qraf_cuda_comm_handle": (i32, [vp, vp]),
        "qraf_cuda_comm_open": (i32, [vp, vp]),
        "qraf_cuda_comm_open_local": (i32, [C.POINTER(vp), i32]),
        "qraf_cuda_comm_destroy": (i32, [vp]),
        "qraf_cuda_matvec_q_sharded": (i32, [vp, W, u32, u32, vp, u32, i32, vp, C.POINTER(vp)]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    return lib


_LIB = None


def _get_lib() -> C.CDLL:
    """The loaded libqraf_cuda.so; raises ImportError when it has not been built."""
    global _LIB
    if _LIB is None:
        _LIB = _load()
    return _LIB


def __getattr__(name):
    if name == "lib":
        return _get_lib()
    raise AttributeError(name)


def last_error() -> str:
    buf = C.create_string_buffer(512)
    _get_lib().qraf_cuda_last_error(buf, len(buf))
    return buf.value.decode(errors="replace")


def check(rc: int) -> None:
    if rc != OK:
        raise QrafError(rc, last_error())


def row_bytes(dtype: int, cols: int, block_size: int = 32) -> int:
    return int(_get_lib().qraf_row_bytes(dtype, block_size, cols))


def fill_normal(seed: int, mean: float, std: float, n: int) -> np.ndarray:
    """std::mt19937(seed) + std::normal_distribution<float>(mean, std), the reference's seeding idiom."""
    out = np.empty(n, dtype=np.float32)
    _get_lib().qraf_fill_normal(seed, mean, std, out.ctypes.data_as(C.POINTER(C.c_float)), n)
    return out


# ── device side (torch tensors as device memory) ─────────────────────────
_TORCH = None


def _torch():
    global _TORCH
    if _TORCH is None:
        import torch

        _TORCH = torch
    return _TORCH


def _stream(stream) -> C.c_void_p:
    torch = _torch()
    if stream is None:
        stream = torch.cuda.current_stream()
    return C.c_void_p(stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream))


def init(device: int = 0) -> None:
    check(_get_lib().qraf_cuda_init(device))


def device_status(clear: bool = True) -> int:
    return int(_get_lib().qraf_cuda_device_status(1 if clear else 0))


class Weight:
    """A quantized [rows][cols] weight in the reference's native block layout on one device."""

    def __init__(self, desc: qraf_weight_t, keepalive=None):
        self.desc = desc
        self._keep = keepalive

    @classmethod
    def from_device(cls, data, dtype: int, rows: int, cols: int, block_size: int = 32) -> "Weight":
        """Wrap a CUDA uint8 tensor holding rows * row_bytes native bytes (no copy)."""
        d = qraf_weight_t()
        check(_get_lib().qraf_cuda_weight_wrap(C.c_void_p(data.data_ptr()), data.numel() * data.element_size(), dtype,
                                        block_size, rows, cols, C.byref(d)))
        return cls(d, keepalive=data)

    @classmethod
    def upload(cls, host: np.ndarray, dtype: int, rows: int, cols: int, block_size: int = 32) -> "Weight":
        host = np.ascontiguousarray(host, dtype=np.uint8)
        d = qraf_weight_t()
        check(_get_lib().qraf_cuda_weight_upload(host.ctypes.data_as(C.c_void_p), host.nbytes, dtype, block_size, rows,
                                          cols, C.byref(d)))
        return cls(d)

    def shard(self, world: int, rank: int) -> "Weight":
        d = qraf_weight_t()
        check(_get_lib().qraf_cuda_weight_shard(C.byref(self.desc), world, rank, C.byref(d)))
        return Weight(d, keepalive=self)

    @property
    def rows(self) -> int:
        return self.desc.rows

    @property
    def cols(self) -> int:
        return self.desc.cols

    @property
    def dtype(self) -> int:
        return self.desc.dtype

    @property
    def nbytes(self) -> int:
        return self.desc.bytes

    def free(self) -> None:
        if self.desc.owned:
            check(_get_lib().qraf_cuda_weight_free(C.byref(self.desc)))

    def __del__(self):
        try:
            if self.desc.owned and self.desc.data:
                _get_lib().qraf_cuda_weight_free(C.byref(self.desc))
        except Exception:
            pass


class DeviceModel:
    """A .qraf file with its Q8_0 / Q4_0 tensors resident on the current device
    (qraf_cuda_model_open: one allocation, the file's bytes unchanged)."""

    def __init__(self, path: str, f32: bool = False):
        h = C.c_void_p()
        check(_get_lib().qraf_cuda_model_open_ex(os.fsencode(path), MODEL_F32 if f32 else 0, C.byref(h)))
        self._h = h

    def tensor_f32(self, name: str):
        """(device address, element count) of an F32 tensor (a model opened with f32=True)."""
        p, n = C.c_void_p(), C.c_uint64()
        check(_get_lib().qraf_cuda_model_tensor_f32(self._h, name.encode(), C.byref(p), C.byref(n)))
        return p.value, n.value

    @property
    def names(self) -> list:
        """Quantized tensors in directory order."""
        lib, out = _get_lib(), []
        while True:
            n = lib.qraf_cuda_model_weight_name(self._h, len(out))
            if n is None:
                return out
            out.append(n.decode())

    def info(self) -> dict:
        n, b, d = C.c_uint32(), C.c_uint64(), C.c_int()
        check(_get_lib().qraf_cuda_model_info(self._h, C.byref(n), C.byref(b), C.byref(d)))
        return {"num_weights": n.value, "device_bytes": b.value, "device": d.value}

    def weight(self, name: str) -> Weight:
        d = qraf_weight_t()
        check(_get_lib().qraf_cuda_model_weight(self._h, name.encode(), C.byref(d)))
        return Weight(d, keepalive=self)

    def config_u32(self, key: str) -> int:
        """Raw bits of a u32 / f32 config entry."""
        v = C.c_uint32()
        check(_get_lib().qraf_cuda_model_config_u32(self._h, key.encode(), C.byref(v)))
        return v.value

    def close(self) -> None:
        if self._h:
            h, self._h = self._h, C.c_void_p()
            check(_get_lib().qraf_cuda_model_close(h))

    def __del__(self):
        try:
            if self._h:
                _get_lib().qraf_cuda_model_close(self._h)
        except Exception:
            pass


def launch_count() -> int:
    """Kernels the library has launched in this process (a captured launch counts once)."""
    return int(_get_lib().qraf_cuda_launch_count())


class Decoder:
    """A Llama / Qwen2 decode engine over a .qraf file (qraf_cuda_decoder_*):
    step() runs one decode step for M slots at once, each with its own KV cache."""

    def __init__(self, path: str, max_slots: int = 1, max_seq: int = 2048, kv_int8: bool = False):
        h = C.c_void_p()
        check(_get_lib().qraf_cuda_decoder_open_ex(os.fsencode(path), max_slots, max_seq,
                                                   DECODER_KV_INT8 if kv_int8 else 0, C.byref(h)))
        self.kv_int8 = kv_int8
        self._h = h
        v, hd, l, ms, mq = (C.c_uint32() for _ in range(5))
        check(_get_lib().qraf_cuda_decoder_info(h, C.byref(v), C.byref(hd), C.byref(l), C.byref(ms), C.byref(mq)))
        self._caches = weakref.WeakSet()   # views of its cache
        self.vocab, self.hidden, self.layers = v.value, hd.value, l.value
        self.max_slots, self.max_seq = ms.value, mq.value

    def step(self, tokens, positions, slots, mode: int = MODE_AUTO, logits=None, stream=None):
        """tokens, positions, slots: contiguous CUDA int32 tensors of M; returns logits [M, vocab]."""
        torch = _torch()
        m = tokens.numel()
        for t in (tokens, positions, slots):
            if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous() or t.numel() != m:
                raise ValueError("tokens, positions and slots must be contiguous CUDA int32 tensors of one length")
        if logits is None:
            logits = torch.empty((m, self.vocab), dtype=torch.float32, device=tokens.device)
        check(_get_lib().qraf_cuda_decoder_step(self._h, m, C.c_void_p(tokens.data_ptr()),
                                                C.c_void_p(positions.data_ptr()), C.c_void_p(slots.data_ptr()),
                                                C.c_void_p(logits.data_ptr()), mode, _stream(stream)))
        return logits

    def step_runs(self, tokens, slots, starts, cu=None, mode: int = MODE_AUTO, logits=None, stream=None):
        """One step over runs of tokens, e.g. prompts or drafts to be verified
        (qraf_cuda_decoder_step_runs; a decoder opened with kv_int8): tokens cu[b] .. cu[b + 1] go to
        positions starts[b] .. of slot slots[b] (without cu, one token each); at most max_slots
        tokens.  tokens, slots, starts, cu: contiguous CUDA int32 tensors.  Returns logits [n, vocab]."""
        n, index = tokens.numel(), tokens.get_device()
        if index < 0:
            raise ValueError("tokens must be a CUDA tensor")
        slots_p, starts_p, cu_p, count = _runs_of(slots, starts, cu, n, index, "starts")
        tokens_p = _ints(tokens, index, "tokens")
        if logits is None:
            logits = _empty((n, self.vocab), _torch().float32, tokens, stream)
        elif logits.dtype != _torch().float32 or logits.get_device() != index or tuple(logits.shape) != (n, self.vocab) or \
                not logits.is_contiguous():
            raise ValueError(f"logits must be a contiguous float32 tensor [{n}, {self.vocab}] on cuda:{index}")
        check(_get_lib().qraf_cuda_decoder_step_runs(self._h, n, tokens_p, slots_p, starts_p, cu_p, count, logits.data_ptr(),
                                                     mode, _stream_on(stream, index)))
        return logits

    def share_prefix(self, slot: int, length: int) -> None:
        """Share the first `length` positions of `slot` among all sequences of the steps over runs
        (qraf_cuda_decoder_share_prefix); 0: no longer."""
        check(_get_lib().qraf_cuda_decoder_share_prefix(self._h, slot, length))

    def layer_cache(self, layer: int) -> "KvCache":
        """One layer of the int8 cache for kv_store, kv_load and kv_attention; it keeps the decoder, until
        that is closed: the operators then refuse it, and tensors taken from it must not be used."""
        d = qraf_kv_t()
        check(_get_lib().qraf_cuda_decoder_kv(self._h, layer, C.byref(d)))
        cache = KvCache._of_desc(d, self)
        self._caches.add(cache)
        return cache

    def kv_read(self, slot: int, layer: int, pos: int, kv_heads: int, head_dim: int):
        """One cache row: (k, v) float32 [kv_heads * head_dim], or with the int8 cache
        (k codes, v codes, k scales, v scales)."""
        n = kv_heads * head_dim
        if self.kv_int8:
            k, v = np.empty(n, np.int8), np.empty(n, np.int8)
            ks, vs = np.empty(kv_heads, np.float32), np.empty(kv_heads, np.float32)
            check(_get_lib().qraf_cuda_decoder_kv_read(self._h, slot, layer, pos, k.ctypes.data, v.ctypes.data,
                                                       ks.ctypes.data_as(C.POINTER(C.c_float)),
                                                       vs.ctypes.data_as(C.POINTER(C.c_float))))
            return k, v, ks, vs
        k, v = np.empty(n, np.float32), np.empty(n, np.float32)
        check(_get_lib().qraf_cuda_decoder_kv_read(self._h, slot, layer, pos, k.ctypes.data, v.ctypes.data, None, None))
        return k, v

    def close(self) -> None:
        if self._h:
            h, self._h = self._h, C.c_void_p()
            for cache in self._caches:
                cache._detach()
            check(_get_lib().qraf_cuda_decoder_close(h))

    def __del__(self):
        try:
            if self._h:
                _get_lib().qraf_cuda_decoder_close(self._h)
        except Exception:
            pass


def host_cache_add(w_host: np.ndarray, dtype: int, rows: int, cols: int, block_size: int = 32) -> None:
    """Preload a host weight into the cache qraf_cuda_matvec_q_host (dispatch_matvec_q) looks up."""
    check(_get_lib().qraf_cuda_host_cache_add(w_host.ctypes.data, w_host.nbytes, dtype, block_size, rows, cols))


def host_cache_info() -> tuple:
    """(entries, device bytes) of that cache."""
    n, b = C.c_uint32(), C.c_uint64()
    check(_get_lib().qraf_cuda_host_cache_info(C.byref(n), C.byref(b)))
    return n.value, b.value


def matvec_q(w: Weight, x, y=None, mode: int = MODE_AUTO, stream=None):
    """Y[m] = dispatch_matvec_q(W, X[m]) on the GPU.  x: CUDA fp32 [M, cols] or [cols]."""
    torch = _torch()
    squeeze = x.dim() == 1
    x2 = x.reshape(1, -1) if squeeze else x
    if x2.dtype != torch.float32 or not x2.is_cuda or not x2.is_contiguous():
        raise ValueError("x must be a contiguous CUDA float32 tensor")
    m = x2.shape[0]
    if x2.shape[1] != w.cols:
        raise ValueError(f"x has {x2.shape[1]} columns, the weight has {w.cols}")
    if y is None:
        y = torch.empty((m, w.rows), dtype=torch.float32, device=x.device)
    check(_get_lib().qraf_cuda_matvec_q(C.byref(w.desc), C.c_void_p(x2.data_ptr()), C.c_void_p(y.data_ptr()), m, mode,
                                 _stream(stream)))
    return y.reshape(w.rows) if squeeze else y


MULTI_MAX_WEIGHTS = 4


def matvec_q_multi(weights, x, ys=None, mode: int = MODE_AUTO, stream=None, norm_w=None, norm_eps: float = 1e-6,
                   biases=None):
    """[W_i X for each weight] in one launch (qraf_cuda_matvec_q_multi): projections of
    the same activations, e.g. a layer's Q, K and V, or gate and up.  Returns the list
    of outputs ([M, rows_i] each, or [rows_i] for a 1-D x).  norm_w: RMSNorm of x
    first; biases: per-weight bias tensors (or None entries) added to the outputs
    (qraf_cuda_matvec_q_multi_ex)."""
    torch = _torch()
    if not 1 <= len(weights) <= MULTI_MAX_WEIGHTS:
        raise ValueError(f"1 to {MULTI_MAX_WEIGHTS} weights")
    squeeze = x.dim() == 1
    x2 = x.reshape(1, -1) if squeeze else x
    if x2.dtype != torch.float32 or not x2.is_cuda or not x2.is_contiguous():
        raise ValueError("x must be a contiguous CUDA float32 tensor")
    m = x2.shape[0]
    if ys is None:
        ys = [torch.empty((m, w.rows), dtype=torch.float32, device=x.device) for w in weights]
    descs = (qraf_weight_t * len(weights))(*[w.desc for w in weights])
    outs = (C.c_void_p * len(weights))(*[y.data_ptr() for y in ys])
    if norm_w is None and biases is None:
        check(_get_lib().qraf_cuda_matvec_q_multi(descs, len(weights), C.c_void_p(x2.data_ptr()), outs, m, mode,
                                                  _stream(stream)))
    else:
        bs = None
        if biases is not None:
            bs = (C.c_void_p * len(weights))(*[b.data_ptr() if b is not None else None for b in biases])
        check(_get_lib().qraf_cuda_matvec_q_multi_ex(
            descs, len(weights), C.c_void_p(x2.data_ptr()), C.c_void_p(norm_w.data_ptr() if norm_w is not None else 0),
            norm_eps, bs, outs, m, mode, _stream(stream)))
    return [y.reshape(w.rows) for y, w in zip(ys, weights)] if squeeze else ys


def matvec_q_swiglu(gate: Weight, up: Weight, x, h=None, mode: int = MODE_AUTO, stream=None, norm_w=None,
                    norm_eps: float = 1e-6):
    """silu(W_gate X) * (W_up X) (qraf_cuda_matvec_q_swiglu): one launch in FAST / AUTO
    for one or two vectors.  Returns [M, rows] (or [rows] for a 1-D x)."""
    torch = _torch()
    squeeze = x.dim() == 1
    x2 = x.reshape(1, -1) if squeeze else x
    if x2.dtype != torch.float32 or not x2.is_cuda or not x2.is_contiguous():
        raise ValueError("x must be a contiguous CUDA float32 tensor")
    m = x2.shape[0]
    if h is None:
        h = torch.empty((m, gate.rows), dtype=torch.float32, device=x.device)
    if norm_w is None:
        check(_get_lib().qraf_cuda_matvec_q_swiglu(C.byref(gate.desc), C.byref(up.desc), C.c_void_p(x2.data_ptr()),
                                                   C.c_void_p(h.data_ptr()), m, mode, _stream(stream)))
    else:
        check(_get_lib().qraf_cuda_matvec_q_swiglu_ex(C.byref(gate.desc), C.byref(up.desc),
                                                      C.c_void_p(x2.data_ptr()), C.c_void_p(norm_w.data_ptr()),
                                                      norm_eps, C.c_void_p(h.data_ptr()), m, mode, _stream(stream)))
    return h.reshape(gate.rows) if squeeze else h


def dot_q(dtype: int, q, x, count: int, block_size: int = 32, mode: int = MODE_EXACT, stream=None):
    """dot_q8_0_f32 / dot_q4_0_f32 on device buffers; returns a 1-element CUDA tensor."""
    torch = _torch()
    out = torch.empty(1, dtype=torch.float32, device=x.device)
    check(_get_lib().qraf_cuda_dot_q(dtype, C.c_void_p(q.data_ptr()), C.c_void_p(x.data_ptr()), count, block_size,
                              C.c_void_p(out.data_ptr()), mode, _stream(stream)))
    return out


def dot_q8_0_f32(q, x, count: int, block_size: int = 32, mode: int = MODE_EXACT):
    return dot_q(Q8_0, q, x, count, block_size, mode)


def dot_q4_0_f32(q, x, count: int, block_size: int = 32, mode: int = MODE_EXACT):
    return dot_q(Q4_0, q, x, count, block_size, mode)


def block_partials(w: Weight, x, stream=None):
    torch = _torch()
    nb = (w.cols + w.desc.block_size - 1) // w.desc.block_size
    out = torch.empty((w.rows, nb), dtype=torch.float32, device=x.device)
    check(_get_lib().qraf_cuda_block_partials(C.byref(w.desc), C.c_void_p(x.data_ptr()), C.c_void_p(out.data_ptr()),
                                       _stream(stream)))
    return out


def limb_partials(w: Weight, x, stream=None):
    """(D [rows][cols/32][4] int32, c [cols/32] fp32): the FAST kernels' per-block integer partial sums for x."""
    torch = _torch()
    nb = w.cols // 32
    d = torch.empty((w.rows, nb, 4), dtype=torch.int32, device=x.device)
    c = torch.empty(nb, dtype=torch.float32, device=x.device)
    check(_get_lib().qraf_cuda_limb_partials(C.byref(w.desc), C.c_void_p(x.data_ptr()), C.c_void_p(d.data_ptr()),
                                              C.c_void_p(c.data_ptr()), _stream(stream)))
    return d, c


def quantize(dtype: int, x, block_size: int = 32, stream=None):
    """quantize_q8_0 / quantize_q4_0 of a contiguous CUDA fp32 tensor (all elements as one sequence)."""
    torch = _torch()
    n = x.numel()
    out = torch.empty(row_bytes(dtype, n, block_size), dtype=torch.uint8, device=x.device)
    check(_get_lib().qraf_cuda_quantize(dtype, C.c_void_p(x.data_ptr()), n, block_size, C.c_void_p(out.data_ptr()),
                                 _stream(stream)))
    return out


def quantize_q8_0(x, block_size: int = 32):
    return quantize(Q8_0, x, block_size)


def quantize_q4_0(x, block_size: int = 32):
    return quantize(Q4_0, x, block_size)


def quantize_rows(dtype: int, x2d, block_size: int = 32, stream=None):
    """Quantize each row of a [rows, cols] CUDA fp32 tensor; returns uint8 [rows, row_bytes]."""
    torch = _torch()
    rows, cols = x2d.shape
    out = torch.empty((rows, row_bytes(dtype, cols, block_size)), dtype=torch.uint8, device=x2d.device)
    check(_get_lib().qraf_cuda_quantize_rows(dtype, C.c_void_p(x2d.data_ptr()), rows, cols, block_size,
                                      C.c_void_p(out.data_ptr()), _stream(stream)))
    return out


def dequantize(dtype: int, q, count: int, block_size: int = 32, stream=None):
    torch = _torch()
    out = torch.empty(count, dtype=torch.float32, device=q.device)
    check(_get_lib().qraf_cuda_dequantize(dtype, C.c_void_p(q.data_ptr()), count, block_size, C.c_void_p(out.data_ptr()),
                                   _stream(stream)))
    return out


# ── KV-cache operators ───────────────────────────────────────────────────
TYPE_F32 = 0
TYPE_F16 = 1
TYPE_BF16 = 2


def _type_of(dtype) -> int:
    global _TYPES
    if _TYPES is None:
        torch = _torch()
        _TYPES = {torch.float32: TYPE_F32, torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16}
    t = _TYPES.get(dtype)
    if t is None:
        raise ValueError(f"{dtype}: float32, float16 or bfloat16")
    return t


_TYPES = None


def _ints(t, index: int, name: str) -> int:
    """Address of a contiguous int32 tensor on device `index`."""
    if t.dtype != _torch().int32 or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor on cuda:{index}")
    return t.data_ptr()


def _runs_of(slots, firsts, cu, n: int, index: int, firsts_name: str) -> tuple:
    """(slots, firsts, cu, number of runs) for the library, checked."""
    count = slots.numel()
    if firsts.numel() != count:
        raise ValueError(f"{count} slots and {firsts.numel()} {firsts_name}")
    if cu is None:
        if count != n:
            raise ValueError(f"{count} slots and {n} rows: without cu each row is a run")
    elif cu.numel() != count + 1:
        raise ValueError(f"cu needs {count + 1} values, has {cu.numel()}")
    return (_ints(slots, index, "slots"), _ints(firsts, index, firsts_name),
            None if cu is None else _ints(cu, index, "cu"), count)


def _rows_of(t, heads: int, dim: int, index: int, name: str) -> tuple:
    """(rows, elements from row to row) of [n, heads, dim] or [n, heads * dim] with contiguous rows."""
    if t.get_device() != index:
        raise ValueError(f"{name} must be on cuda:{index}")
    shape, width = t.shape, heads * dim
    d = len(shape)
    if not (d == 3 and shape[1] == heads and shape[2] == dim or d == 2 and shape[1] == width):
        raise ValueError(f"{name} must be [n, {heads}, {dim}] or [n, {width}], is {list(shape)}")
    if t.is_contiguous():
        return shape[0], width
    stride = t.stride()
    if (dim if d == 3 else width) > 1 and stride[-1] != 1 or d == 3 and heads > 1 and stride[1] != dim:
        raise ValueError(f"{name}: the values of a row must be contiguous")
    if shape[0] <= 1:
        return shape[0], width
    if stride[0] < width:
        raise ValueError(f"{name}: rows overlap")
    return shape[0], stride[0]


def _allocating_on(stream, device):
    """Where what a call allocates belongs to the stream it runs on: memory that the current
    stream has just let go may still be in use there."""
    torch = _torch()
    return torch.cuda.stream(stream if hasattr(stream, "cuda_stream") else
                             torch.cuda.ExternalStream(int(stream), device=device))


def _empty(shape, dtype, like, stream):
    """A tensor on `like`'s device for a call on `stream`."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with _allocating_on(stream, like.device):
        return like.new_empty(shape, dtype=dtype)


def _stream_on(stream, index: int):
    """The stream's handle; the current stream of device `index` when it is None."""
    if stream is None:
        return _torch()._C._cuda_getCurrentRawStream(index)
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


class KvCache:
    """The int8 KV cache of one layer: row r of slot s holds, per KV head, head_dim
    int8 codes of K and of V and one fp32 scale of each (the reference's
    QuantizedKVCache layout); a value is code * scale.

    k, v: int8 [slots, rows, kv_heads, head_dim]; k_scale, v_scale: float32
    [slots, rows, kv_heads], all on one device.  Slots may lie further apart than
    their rows (a view of a larger tensor), by the same number of rows in all four."""

    def __init__(self, slots: int, rows: int, kv_heads: int, head_dim: int, device=None):
        torch = _torch()
        shape = (slots, rows, kv_heads)
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        self._set(*(torch.zeros(*shape, head_dim, dtype=torch.int8, device=dev) for _ in range(2)),
                  *(torch.zeros(shape, dtype=torch.float32, device=dev) for _ in range(2)))

    @classmethod
    def from_tensors(cls, k, v, k_scale, v_scale) -> "KvCache":
        """A cache in the caller's tensors (nothing is copied)."""
        self = cls.__new__(cls)
        self._set(k, v, k_scale, v_scale)
        return self

    def _set(self, k, v, k_scale, v_scale) -> None:
        torch = _torch()
        if k.dim() != 4 or k.dtype != torch.int8 or v.dtype != torch.int8 or v.shape != k.shape:
            raise ValueError("k and v must be int8 tensors of one shape [slots, rows, kv_heads, head_dim]")
        if any(s.shape != k.shape[:3] or s.dtype != torch.float32 for s in (k_scale, v_scale)):
            raise ValueError("k_scale and v_scale must be float32 [slots, rows, kv_heads]")
        if any(not t.is_cuda or t.device != k.device for t in (k, v, k_scale, v_scale)):
            raise ValueError("the cache's tensors must be on one CUDA device")
        slots, rows, heads, dim = k.shape
        if 0 in k.shape:
            raise ValueError("the cache is empty")
        apart = set()
        for t, width in ((k, heads * dim), (v, heads * dim), (k_scale, heads), (v_scale, heads)):
            if not t[0].is_contiguous():
                raise ValueError("the rows of a slot must be contiguous")
            if slots > 1:
                if t.stride(0) % width:
                    raise ValueError("slots must lie a whole number of rows apart")
                apart.add(t.stride(0) // width)
        if len(apart) > 1:
            raise ValueError("codes and scales must have their slots the same number of rows apart")
        d = qraf_kv_t()
        check(_get_lib().qraf_cuda_kv_wrap(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), slots,
                                           rows, apart.pop() if apart else rows, heads, dim, C.byref(d)))
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self._describe(d)

    @classmethod
    def _of_desc(cls, d: qraf_kv_t, keepalive) -> "KvCache":
        """A cache in the library's memory: its tensors are views of that."""
        torch = _torch()
        self = cls.__new__(cls)
        self._keep = keepalive
        for name, typestr, size in (("k", "|i1", 1), ("v", "|i1", 1), ("k_scale", "<f4", 4), ("v_scale", "<f4", 4)):
            shape = (d.slots, d.rows, d.kv_heads) + ((d.head_dim,) if size == 1 else ())
            width = d.head_dim if size == 1 else 1   # elements of a (row, head)
            strides = (d.slot_rows * d.kv_heads * width * size, d.kv_heads * width * size, width * size) + ((1,) if size == 1 else ())

            class _Holder:
                __cuda_array_interface__ = {"shape": shape, "typestr": typestr, "data": (getattr(d, name), False), "version": 3,
                                            "strides": strides}
                owner = keepalive   # the tensor keeps this object

            setattr(self, name, torch.as_tensor(_Holder(), device=f"cuda:{d.device}"))
        self._describe(d)
        return self

    def _describe(self, d: qraf_kv_t) -> None:
        self.desc = d
        self.device, self._index = self.k.device, d.device
        self.slots, self.rows, self.kv_heads, self.head_dim = d.slots, d.rows, d.kv_heads, d.head_dim
        self._workspace = {}

    @property
    def _ref(self):
        """The descriptor for a call of the library."""
        if not self.desc.k:
            raise ValueError("the decoder of this cache is closed")
        return C.byref(self.desc)

    def _detach(self) -> None:
        """The memory behind the cache goes away."""
        C.memset(C.byref(self.desc), 0, C.sizeof(self.desc))
        self.k = self.v = self.k_scale = self.v_scale = None


def kv_store(cache: KvCache, k, v, slots, starts, cu=None, stream=None) -> None:
    """Quantise rows of K and V into `cache` as they are written (qraf_cuda_kv_store).

    k, v: float32, float16 or bfloat16 [n, kv_heads, head_dim] (or [n, kv_heads * head_dim]),
    rows contiguous, any stride between them.  Rows cu[b] .. cu[b + 1] go to rows starts[b] ..
    of slot slots[b] (int32 CUDA tensors; without cu, one row each); slot -1 and rows behind
    the last run are left out, and where two runs write one row the later one stays."""
    ref, heads, dim, index = cache._ref, cache.kv_heads, cache.head_dim, cache._index
    n, ld_k = _rows_of(k, heads, dim, index, "k")
    m, ld_v = _rows_of(v, heads, dim, index, "v")
    if m != n or v.dtype != k.dtype:
        raise ValueError("k and v must have one type and length")
    slots_p, starts_p, cu_p, count = _runs_of(slots, starts, cu, n, index, "starts")
    check(_get_lib().qraf_cuda_kv_store(ref, k.data_ptr(), v.data_ptr(), _type_of(k.dtype), ld_k, ld_v, n, slots_p,
                                        starts_p, cu_p, count, _stream_on(stream, index)))


def kv_load(cache: KvCache, slots, starts, cu=None, n=None, dtype=None, k=None, v=None, stream=None) -> tuple:
    """Rows of K and V read back as numbers (qraf_cuda_kv_load), the runs as in kv_store.

    n: the number of rows (needed with cu, unless k and v are given to be written);
    dtype: float32 (default), float16 or bfloat16.  Returns (k, v) [n, kv_heads, head_dim]."""
    ref, heads, dim, index = cache._ref, cache.kv_heads, cache.head_dim, cache._index
    if (k is None) != (v is None):
        raise ValueError("k and v go together")
    if k is None:
        n = slots.numel() if n is None and cu is None else n
        if n is None:
            raise ValueError("n, the number of rows, is needed with cu")
        dtype = _torch().float32 if dtype is None else dtype
        k, v = (_empty((n, heads, dim), dtype, cache.k, stream) for _ in range(2))
        ld_k = ld_v = heads * dim
    else:
        n, ld_k = _rows_of(k, heads, dim, index, "k")
        m, ld_v = _rows_of(v, heads, dim, index, "v")
        if m != n or v.dtype != k.dtype:
            raise ValueError("k and v must have one type and length")
    slots_p, starts_p, cu_p, count = _runs_of(slots, starts, cu, n, index, "starts")
    check(_get_lib().qraf_cuda_kv_load(ref, k.data_ptr(), v.data_ptr(), _type_of(k.dtype), ld_k, ld_v, n, slots_p,
                                       starts_p, cu_p, count, _stream_on(stream, index)))
    return k, v


def kv_attention(q, cache: KvCache, slots, lens, cu=None, prefix=None, prefix_slot: int = 0, prefix_len: int = 0,
                 max_len=None, scale=None, out=None, stream=None):
    """Attention of new tokens over the int8 cache, behind a prefix that the whole batch
    shares (qraf_cuda_kv_attention).

    q: float32, float16 or bfloat16 [n, heads, head_dim] (or [n, heads * head_dim]), heads a
    multiple of the cache's kv_heads.  Tokens cu[b] .. cu[b + 1] are sequence b's new ones
    (without cu, one each); its slot slots[b] holds lens[b] rows, theirs included, and token
    i of m sees the first lens[b] - m + 1 + i of them after the prefix_len rows of slot
    prefix_slot of the KvCache `prefix`.  A token that sees nothing gets zeros; tokens of
    slot -1 or behind the last sequence keep what `out` holds.  max_len: no lens[b] is larger
    (default: the cache's rows).  scale: default head_dim ** -0.5.  Weights are exact to 22 bits of
    themselves or 2^-31 of the largest V scale that the row sees.  Returns out, shaped like q."""
    ref, dim, index = cache._ref, cache.head_dim, cache._index
    if q.dim() not in (2, 3):
        raise ValueError("q must be [n, heads, head_dim] or [n, heads * head_dim]")
    heads = q.shape[1] if q.dim() == 3 else q.shape[1] // dim
    n, q_ld = _rows_of(q, heads, dim, index, "q")
    if out is None:
        out, out_ld = _empty(q.shape, q.dtype, q, stream), heads * dim
    else:
        m, out_ld = _rows_of(out, heads, dim, index, "out")
        if m != n or out.dtype != q.dtype:
            raise ValueError("out must have q's type and length")
    slots_p, lens_p, cu_p, count = _runs_of(slots, lens, cu, n, index, "lens")
    if prefix_len < 0 or prefix_slot < 0:
        raise ValueError("prefix_len and prefix_slot cannot be negative")
    if prefix_len and prefix is None:
        raise ValueError("prefix_len without a prefix")
    max_len = cache.rows if max_len is None else max_len
    if max_len < 0:
        raise ValueError("max_len cannot be negative")
    lib = _get_lib()
    key = (prefix_len, n, heads, count, cu is None, max_len)
    size = cache._workspace.get(key)
    if size is None:   # bytes by shape; the memory itself belongs to the call
        b = C.c_uint64()
        check(lib.qraf_cuda_kv_attention_workspace(ref, prefix_len, n, heads, count, cu is not None, max_len,
                                                   C.byref(b)))
        if len(cache._workspace) > 4096:
            cache._workspace.clear()
        size = cache._workspace[key] = b.value
    ws = _empty(size, _torch().uint8, q, stream) if size else None
    check(lib.qraf_cuda_kv_attention(ref, prefix._ref if prefix_len else None, prefix_slot, prefix_len, q.data_ptr(),
                                     out.data_ptr(), _type_of(q.dtype), q_ld, out_ld, n, heads, slots_p, lens_p, cu_p, count,
                                     max_len, dim ** -0.5 if scale is None else scale, ws.data_ptr() if size else None, size,
                                     _stream_on(stream, index)))
    return out


# ── from logits to accepted tokens ───────────────────────────────────────
def token_probs(logits, temperature: float = 1.0, out=None, stream=None):
    """softmax(logits / temperature) over the last dimension (qraf_cuda_token_probs) of a
    float32 CUDA tensor [rows, vocab] or [vocab]; -inf gives 0, a row of nothing else
    zeros.  out may be logits itself."""
    torch = _torch()
    x = logits.reshape(1, -1) if logits.dim() == 1 else logits
    index = x.get_device()
    if x.dim() != 2 or x.dtype != torch.float32 or index < 0:
        raise ValueError("logits must be a CUDA float32 tensor [rows, vocab]")
    rows, vocab = x.shape
    _, x_ld = _rows_of(x, 1, vocab, index, "logits")
    _check_current(index)
    if out is None:
        out, y_ld = _empty(logits.shape, torch.float32, x, stream), vocab
    else:
        y = out.reshape(1, -1) if out.dim() == 1 else out
        m, y_ld = _rows_of(y, 1, vocab, index, "out")
        if m != rows or y.dtype != torch.float32:
            raise ValueError("out must be float32 and shaped like logits")
    check(_get_lib().qraf_cuda_token_probs(x.data_ptr(), x_ld, out.data_ptr(), y_ld, rows, vocab, temperature,
                                           _stream_on(stream, index)))
    return out


def verify_drafts(target, draft, tokens, u, u_last, counts=None, stream=None) -> tuple:
    """Verify drafted tokens against the target's probabilities from given uniform random
    numbers (qraf_cuda_verify_drafts).

    target: float32 [B, K + 1, vocab] probabilities (row i: after the first i drafts); draft:
    float32 [B, K, vocab]; tokens: int32 [B, K]; u: float32 [B, K]; u_last: float32 [B];
    counts: int32 [B], the drafts of each sequence (default K; -1: its outputs are left as
    they were, here uninitialised).  Rows of the vocabulary are contiguous, other strides free.
    Draft i stands while u_i q_i(x_i) < p_i(x_i); the first that falls is replaced by a draw from
    max(p_i - q_i, 0), and when all stand one more token is drawn from the next row.  Returns
    (int32 [B, K + 1]: the standing drafts, the drawn token, then -1; int32 [B]: how many stand)."""
    f32 = _torch().float32
    index = target.get_device()
    if target.dim() != 3:
        raise ValueError("target must be [B, K + 1, vocab]")
    b, k1, vocab = target.shape
    k = k1 - 1
    if k < 0 or draft.shape != (b, k, vocab) or tokens.shape != (b, k) or u.shape != (b, k) or u_last.shape != (b,) or \
            (counts is not None and counts.shape != (b,)):
        raise ValueError(f"shapes do not fit {b} sequences of {k} drafts over {vocab} tokens")
    for t in (target, draft, u, u_last):
        if t.dtype != f32 or t.get_device() != index or index < 0:
            raise ValueError("target, draft, u and u_last must be float32 tensors on one CUDA device")
    if not u.is_contiguous() or not u_last.is_contiguous():
        raise ValueError("u and u_last must be contiguous")
    strides = []
    for t in (target, draft):
        seq, row, one = t.stride()
        if one != 1 and vocab > 1 and t.numel():
            raise ValueError("rows of target and draft must be contiguous")
        # a dimension of one has any stride
        strides += [seq if b > 1 else max(seq, vocab), row if t.shape[1] > 1 else max(row, vocab)]
    _check_current(index)
    counts_p = None if counts is None else _ints(counts, index, "counts")
    i32 = _torch().int32
    out, accepted = _empty((b, k1), i32, target, stream), _empty(b, i32, target, stream)
    check(_get_lib().qraf_cuda_verify_drafts(target.data_ptr(), strides[0], strides[1], draft.data_ptr(), strides[2],
                                             strides[3], _ints(tokens, index, "tokens"), u.data_ptr(), u_last.data_ptr(),
                                             counts_p, b, k, vocab, out.data_ptr(), accepted.data_ptr(),
                                             _stream_on(stream, index)))
    return out, accepted


def _check_current(index: int) -> None:
    current = _torch().cuda.current_device()
    if index != current:
        raise ValueError(f"the tensors are on cuda:{index}, the current device is cuda:{current}")


# ── host side: the reference-facing entry ────────────────────────────────
def dispatch_matvec_q(w_data: np.ndarray, w_size: int, w_dtype: int, block_size: int, out_dim: int, in_dim: int,
                      x: np.ndarray, y: np.ndarray, m: int = 1, mode: int = MODE_EXACT) -> None:
    """qraf::dispatch_matvec_q with host buffers (backend.cpp:131-199); y is overwritten."""
    if not (w_data.flags.c_contiguous and x.flags.c_contiguous and y.flags.c_contiguous):
        raise ValueError("host buffers must be C-contiguous")
    # plain integer addresses: a third of the cost of ctypes.data_as per argument
    check(_get_lib().qraf_cuda_matvec_q_host(w_data.ctypes.data, w_size, w_dtype, block_size, out_dim, in_dim,
                                             x.ctypes.data, y.ctypes.data, m, mode))


def host_cache_clear() -> None:
    check(_get_lib().qraf_cuda_host_cache_clear())


# ── row-sharded matvec over several GPUs ─────────────────────────────────
COMM_HANDLE_BYTES = 512
COMM_BUFFERS = 4


class Comm:
    """One rank's buffers for the fused row-sharded matvec (qraf_cuda_comm_*)."""

    def __init__(self, world: int, rank: int, capacity_floats: int):
        h = C.c_void_p()
        check(_get_lib().qraf_cuda_comm_create(world, rank, capacity_floats, C.byref(h)))
        self.h, self.world, self.rank = h, world, rank

    def handle(self) -> bytes:
        buf = C.create_string_buffer(COMM_HANDLE_BYTES)
        check(_get_lib().qraf_cuda_comm_handle(self.h, buf))
        return buf.raw

    def open(self, all_handles: list[bytes]) -> None:
        blob = b"".join(all_handles)
        check(_get_lib().qraf_cuda_comm_open(self.h, C.create_string_buffer(blob, len(blob))))

    @staticmethod
    def open_local(comms: list["Comm"]) -> None:
        arr = (C.c_void_p * len(comms))(*[c.h for c in comms])
        check(_get_lib().qraf_cuda_comm_open_local(arr, len(comms)))

    def matvec_q(self, shard: Weight, total_rows: int, row_offset: int, x, mode: int = MODE_FAST, stream=None):
        """Rows of `shard` into every rank's y; returns this rank's full y ([M, total_rows], a view)."""
        torch = _torch()
        x2 = x.reshape(1, -1) if x.dim() == 1 else x
        m = x2.shape[0]
        yp = C.c_void_p()
        check(_get_lib().qraf_cuda_matvec_q_sharded(self.h, C.byref(shard.desc), total_rows, row_offset,
                                                    C.c_void_p(x2.data_ptr()), m, mode, _stream(stream), C.byref(yp)))
        return _wrap_device_floats(yp.value, m * total_rows, x.device).view(m, total_rows)

    def destroy(self) -> None:
        if self.h:
            _get_lib().qraf_cuda_comm_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass


def _wrap_device_floats(ptr: int, n: int, device):
    """A torch view of n fp32 values at a device address owned by the library."""
    torch = _torch()

    class _Holder:
        __cuda_array_interface__ = {"shape": (n,), "typestr": "<f4", "data": (ptr, False), "version": 3,
                                    "strides": None}

    return torch.as_tensor(_Holder(), device=device)


def make_comm(world: int, rank: int, capacity_floats: int, all_gather_bytes) -> Comm:
    """Create this rank's Comm and open it, exchanging handles with `all_gather_bytes`
    (a callable taking this rank's bytes and returning every rank's, in rank order)."""
    c = Comm(world, rank, capacity_floats)
    handles = all_gather_bytes(c.handle())
    if len(handles) != world or any(len(h) != COMM_HANDLE_BYTES for h in handles):
        raise QrafError(ERR_COMM, "handle exchange returned the wrong number or size of handles")
    c.open(handles)
    return c


def torch_all_gather_bytes(group=None):
    """all_gather_bytes for make_comm over an initialised torch.distributed group."""
    import torch.distributed as dist

    def gather(b: bytes) -> list[bytes]:
        out = [None] * dist.get_world_size(group)
        dist.all_gather_object(out, b, group=group)
        return out

    return gather
