"""HipBackend: the MathBackend / DeviceBackend methods of the int8 Llama path
(crates/scry-llm/src/backend/mod.rs) over the scry_hip C ABI.

Names and argument meaning follow the reference trait: static methods, owned
storage returned by every op, errors raised (the reference panics).  Storage
lives on the GPU; ``to_vec`` copies back to numpy.
"""
from __future__ import annotations

import ctypes as C
from array import array

import numpy as np

from . import _lib
from ._lib import call, load


_CAPSULE_NEW = C.pythonapi.PyCapsule_New
_CAPSULE_NEW.restype, _CAPSULE_NEW.argtypes = C.py_object, [C.c_void_p, C.c_char_p, C.c_void_p]
_capsule_end = None  # the library's destructor of such capsules, on first use
_device = 0  # the device of init_gpu


def _f32(a) -> np.ndarray:
    return np.ascontiguousarray(a, dtype=np.float32).ravel()


class Storage:
    """Device f32 storage (DeviceBackend::Storage)."""

    __slots__ = ("h", "n")

    def __init__(self, handle: int, n: int):
        self.h = handle
        self.n = n

    def to_vec(self) -> np.ndarray:
        out = np.empty(self.n, np.float32)
        call("scry_hip_to_vec", self.h, out.ctypes.data, self.n)
        return out

    def __dlpack_device__(self) -> tuple[int, int]:
        return 10, _device  # ROCm

    def __dlpack__(self, *, stream=None, max_version=None, dl_device=None, copy=None):
        """The f32 values where they lie on the device, without a copy, for
        torch.from_dlpack and its like (torch imported before this package, so
        that both use one HIP runtime).  stream: what it does next comes after
        the ops called so far (None, 0, 1: the default stream); -1: the caller
        waits, as with HipBackend.synchronize().  Writes through the view, and
        reads that outlive it, are ordered by the caller."""
        if copy or (dl_device is not None and tuple(dl_device) != self.__dlpack_device__()):
            raise BufferError("a storage is viewed where it lies")
        global _capsule_end
        if _capsule_end is None:
            _capsule_end = C.cast(load().scry_hip_dlpack_capsule_end, C.c_void_p)
        m = C.c_void_p()
        call("scry_hip_buf_dlpack", self.h, None if stream in (None, 0, 1, -1) else stream, stream != -1, C.byref(m))
        return _CAPSULE_NEW(m, b"dltensor", _capsule_end)

    def free(self) -> None:
        if self.h:
            load().scry_hip_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class I8Storage:
    """Device int8 weight storage (DeviceBackend::I8Storage)."""

    __slots__ = ("h", "n")

    def __init__(self, handle: int, n: int):
        self.h = handle
        self.n = n

    def to_vec(self) -> np.ndarray:
        out = np.empty(self.n, np.int8)
        call("scry_hip_i8_to_vec", self.h, out.ctypes.data, self.n)
        return out

    def free(self) -> None:
        if self.h:
            load().scry_hip_i8_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class KvCache8:
    """An int8 KV cache of max_seq rows of one layer and one sequence."""

    __slots__ = ("h", "max_seq", "n_kv", "head_dim")

    def __init__(self, handle: int, max_seq: int, n_kv: int, head_dim: int):
        self.h = handle
        self.max_seq = max_seq
        self.n_kv = n_kv
        self.head_dim = head_dim

    def free(self) -> None:
        if self.h:
            load().scry_hip_kv8_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def _out():
    return C.c_void_p()


def _ints(a, dtype=np.int32) -> np.ndarray:
    """A host array of whole numbers, refused where dtype does not hold them."""
    x = np.ascontiguousarray(a)
    if x.dtype != dtype:
        y = x.astype(dtype)
        if (x != y).any():
            raise ValueError(f"expected values that {np.dtype(dtype).name} holds")
        x = y
    return x


def _at(a: np.ndarray) -> int:
    """Where an array's values lie (ndarray.ctypes takes 1 us)."""
    return a.__array_interface__["data"][0]


def _starts(start) -> array:
    """One context length per sequence, as C ints."""
    try:
        if getattr(start, "ndim", 1) == 1:
            return array("i", start)
    except (TypeError, OverflowError):
        pass
    raise ValueError("one context length per sequence, as whole numbers below 2^31")


def _parents(parents, n_seq: int, rows: int):
    """[n_seq, rows] parents, or one tree [rows] that every sequence has."""
    if parents is None:
        return None, None
    a = _ints(parents, np.int64)
    if a.shape == (rows,):
        a = np.ascontiguousarray(np.broadcast_to(a, (n_seq, rows)))
    if a.shape != (n_seq, rows):
        raise ValueError(f"parents must be [{n_seq}, {rows}] or [{rows}]")
    return a, _at(a)


def _handles(items, n_seq: int) -> array:
    if len(items) != n_seq:
        raise ValueError("one cache per sequence")
    return array("Q", [i.h or 0 for i in items])


def _st(h: C.c_void_p, n: int) -> Storage:
    return Storage(h.value, n)


class HipBackend:
    """Static-method backend, mirroring the reference trait surface."""

    # ---- runtime (cuda.rs:39-52 init_gpu, 1193-1197 synchronize)
    @staticmethod
    def init_gpu(device: int = 0) -> None:
        global _device
        call("scry_hip_init", device)
        _device = device

    @staticmethod
    def synchronize() -> None:
        call("scry_hip_synchronize")

    @staticmethod
    def device_info() -> dict:
        name = C.create_string_buffer(256)
        arch = C.create_string_buffer(64)
        cu = C.c_int()
        call("scry_hip_device_info", name, 256, C.byref(cu), arch, 64)
        return {"name": name.value.decode(), "arch": arch.value.decode(), "cu_count": cu.value}

    # ---- DeviceBackend
    @staticmethod
    def zeros(n: int) -> Storage:
        o = _out()
        call("scry_hip_zeros", n, C.byref(o))
        return _st(o, n)

    @staticmethod
    def from_vec(data) -> Storage:
        a = _f32(data)
        o = _out()
        call("scry_hip_from_vec", a.ctypes.data, a.size, C.byref(o))
        return _st(o, a.size)

    @staticmethod
    def init_gpu_bf16(device: int = 0) -> None:
        """init_gpu_bf16 (cuda.rs:55-59): init, then bf16 mode."""
        global _device
        call("scry_hip_init_bf16", device)
        _device = device

    @staticmethod
    def set_bf16_mode(on: bool) -> None:
        call("scry_hip_set_bf16_mode", int(bool(on)))

    @staticmethod
    def bf16_mode() -> bool:
        v = C.c_int()
        call("scry_hip_bf16_mode", C.byref(v))
        return bool(v.value)

    @staticmethod
    def from_vec_with_bf16(data, bf16_bytes) -> Storage:
        """DeviceBackend::from_vec_with_bf16 (mod.rs:28-32): bf16_bytes are the
        little-endian bf16 words of the same values (uint16 array or bytes)."""
        a = _f32(data)
        h = np.frombuffer(bytes(bf16_bytes), np.uint16) if isinstance(bf16_bytes, (bytes, bytearray)) \
            else np.ascontiguousarray(bf16_bytes, np.uint16).ravel()
        if h.size != a.size:
            raise ValueError("from_vec_with_bf16: bf16 data and f32 data differ in length")
        o = _out()
        call("scry_hip_from_vec_with_bf16", a.ctypes.data, h.ctypes.data, a.size, C.byref(o))
        return _st(o, a.size)

    @staticmethod
    def to_vec(s: Storage) -> np.ndarray:
        return s.to_vec()

    @staticmethod
    def clone_storage(s: Storage) -> Storage:
        o = _out()
        call("scry_hip_clone_storage", s.h, C.byref(o))
        return _st(o, s.n)

    @staticmethod
    def i8_from_vec(data) -> I8Storage:
        a = np.ascontiguousarray(data, dtype=np.int8).ravel()
        o = _out()
        call("scry_hip_i8_from_vec", a.ctypes.data, a.size, C.byref(o))
        return I8Storage(o.value, a.size)

    @staticmethod
    def i8_to_vec(s: I8Storage) -> np.ndarray:
        return s.to_vec()

    # ---- quantize.rs on the device
    @staticmethod
    def quantize_symmetric(w: Storage) -> tuple[I8Storage, float]:
        o = _out()
        s = C.c_float()
        call("scry_hip_quantize_symmetric", w.h, C.byref(o), C.byref(s))
        return I8Storage(o.value, w.n), np.float32(s.value)

    @staticmethod
    def dequantize(q: I8Storage, scale: float) -> Storage:
        o = _out()
        call("scry_hip_dequantize", q.h, float(scale), C.byref(o))
        return _st(o, q.n)

    @staticmethod
    def quantize_block32(w: Storage, k: int, n: int) -> tuple[I8Storage, Storage]:
        q, s = _out(), _out()
        call("scry_hip_quantize_block32", w.h, k, n, C.byref(q), C.byref(s))
        return I8Storage(q.value, w.n), _st(s, n * ((k + 31) // 32))

    # ---- MathBackend int8 (mod.rs:520-557)
    @staticmethod
    def matmul_i8_f32(a: Storage, b_q: I8Storage, scale: float, m: int, k: int, n: int) -> Storage:
        o = _out()
        call("scry_hip_matmul_i8_f32", a.h, b_q.h, float(scale), m, k, n, C.byref(o))
        return _st(o, m * n)

    @staticmethod
    def matmul_i8_f32_bias(a, b_q, scale, bias: Storage, m, k, n) -> Storage:
        o = _out()
        call("scry_hip_matmul_i8_f32_bias", a.h, b_q.h, float(scale), bias.h, m, k, n, C.byref(o))
        return _st(o, m * n)

    @staticmethod
    def matmul_i8_f32_block32(a, b_q, scales: Storage, m, k, n) -> Storage:
        o = _out()
        call("scry_hip_matmul_i8_f32_block32", a.h, b_q.h, scales.h, m, k, n, C.byref(o))
        return _st(o, m * n)

    # ---- MathBackend glue
    @staticmethod
    def matmul(a, b, m, k, n, trans_a=False, trans_b=False) -> Storage:
        o = _out()
        call("scry_hip_matmul", a.h, b.h, m, k, n, int(trans_a), int(trans_b), C.byref(o))
        return _st(o, m * n)

    @staticmethod
    def matmul_bias(a, b, bias, m, k, n, trans_a=False, trans_b=False) -> Storage:
        """C = A @ B + bias, the bias row [n] added to every row (mod.rs:62-86)."""
        o = _out()
        call("scry_hip_matmul_bias", a.h, b.h, bias.h, m, k, n, int(trans_a), int(trans_b),
             C.byref(o))
        return _st(o, m * n)

    @staticmethod
    def matmul_strided_batched(a, b, batch, m, k, n, trans_a=False, trans_b=False) -> Storage:
        o = _out()
        call("scry_hip_matmul_strided_batched", a.h, b.h, batch, m, k, n, int(trans_a),
             int(trans_b), C.byref(o))
        return _st(o, batch * m * n)

    @staticmethod
    def rmsnorm(x, w, rows, d, eps=1e-5) -> Storage:
        o = _out()
        call("scry_hip_rmsnorm", x.h, w.h, rows, d, float(eps), C.byref(o))
        return _st(o, rows * d)

    @staticmethod
    def rope_with_freqs_preloaded(x, seq, n_heads, head_dim, start_pos, freqs) -> Storage:
        o = _out()
        call("scry_hip_rope_with_freqs_preloaded", x.h, seq, n_heads, head_dim, start_pos,
             freqs.h, C.byref(o))
        return _st(o, x.n)

    @staticmethod
    def rope_with_freqs_scaled_preloaded(x, seq, n_heads, head_dim, start_pos, freqs,
                                         scale) -> Storage:
        o = _out()
        call("scry_hip_rope_with_freqs_scaled_preloaded", x.h, seq, n_heads, head_dim,
             start_pos, freqs.h, float(scale), C.byref(o))
        return _st(o, x.n)

    @staticmethod
    def scale(x, s) -> Storage:
        o = _out()
        call("scry_hip_scale", x.h, float(s), C.byref(o))
        return _st(o, x.n)

    @staticmethod
    def softmax(x, rows, cols) -> Storage:
        o = _out()
        call("scry_hip_softmax", x.h, rows, cols, C.byref(o))
        return _st(o, rows * cols)

    @staticmethod
    def swiglu(gate, up) -> Storage:
        o = _out()
        call("scry_hip_swiglu", gate.h, up.h, C.byref(o))
        return _st(o, gate.n)

    @staticmethod
    def add(a, b) -> Storage:
        o = _out()
        call("scry_hip_add", a.h, b.h, C.byref(o))
        return _st(o, a.n)

    @staticmethod
    def embedding(weight, ids, vocab, dim) -> Storage:
        idx = np.ascontiguousarray(ids, dtype=np.int64).ravel()
        o = _out()
        call("scry_hip_embedding", weight.h, idx.ctypes.data, idx.size, vocab, dim, C.byref(o))
        return _st(o, idx.size * dim)

    @staticmethod
    def gather_reshape_repeat_kv(cache, max_seq, cached_len, n_kv, n_q, head_dim) -> Storage:
        o = _out()
        call("scry_hip_gather_reshape_repeat_kv", cache.h, max_seq, cached_len, n_kv, n_q,
             head_dim, C.byref(o))
        return _st(o, n_q * cached_len * head_dim)

    @staticmethod
    def repeat_kv(x, n_kv, n_q, seq, d_head) -> Storage:
        o = _out()
        call("scry_hip_repeat_kv", x.h, n_kv, n_q, seq, d_head, C.byref(o))
        return _st(o, n_q * seq * d_head)

    @staticmethod
    def scatter_rows(dst, src, total_rows, cols, row_start, row_count) -> None:
        call("scry_hip_scatter_rows", dst.h, src.h, total_rows, cols, row_start, row_count)

    @staticmethod
    def argmax(logits: Storage) -> int:
        out = C.c_int64()
        call("scry_hip_argmax", logits.h, C.byref(out))
        return int(out.value)

    @staticmethod
    def sample_token(logits: Storage, config, rng) -> int:
        """sample_token (generate.rs:92-186) on the device: config is a
        SamplingConfig, rng an Rng whose state advances by the draw."""
        sc = _lib.SamplingConfigC(float(config.temperature), int(config.top_k),
                                  float(config.top_p), int(config.max_tokens))
        st = C.c_uint64(rng.state)
        out = C.c_int64()
        call("scry_hip_sample_token", logits.h, C.byref(sc), C.byref(st), C.byref(out))
        rng.state = int(st.value)
        return int(out.value)

    @staticmethod
    def sample_token_noalloc(logits: Storage, config, rng) -> int:
        """sample_token with no device allocation (a static scratch array per
        GPU, vocabularies up to 262144): same result and rng advance."""
        sc = _lib.SamplingConfigC(float(config.temperature), int(config.top_k),
                                  float(config.top_p), int(config.max_tokens))
        st = C.c_uint64(rng.state)
        out = C.c_int64()
        call("scry_hip_sample_token_noalloc", logits.h, C.byref(sc), C.byref(st), C.byref(out))
        rng.state = int(st.value)
        return int(out.value)

    # ---- the rest of the trait surface (mod.rs; CPU semantics cpu.rs)
    @staticmethod
    def ones(n: int) -> Storage:
        o = _out()
        call("scry_hip_ones", n, C.byref(o))
        return _st(o, n)

    @staticmethod
    def add_shapes(a, a_shape, b, b_shape, out_shape) -> Storage:
        """MathBackend::add with broadcasting (shapes as tuples)."""
        dims = [(C.c_size_t * len(d))(*d) for d in (a_shape, b_shape, out_shape)]
        o = _out()
        call("scry_hip_add_broadcast", a.h, dims[0], len(a_shape), b.h, dims[1], len(b_shape),
             dims[2], len(out_shape), C.byref(o))
        return _st(o, int(np.prod(out_shape)))

    @staticmethod
    def add_inplace(dst, src) -> None:
        call("scry_hip_add_inplace", dst.h, src.h)

    @staticmethod
    def scaled_softmax(x, scale, rows, cols) -> Storage:
        o = _out()
        call("scry_hip_scaled_softmax", x.h, scale, rows, cols, C.byref(o))
        return _st(o, x.n)

    @staticmethod
    def layernorm(x, gamma, beta, rows, d, eps=1e-5):
        """Returns (output, mean [rows], rstd [rows])."""
        o, mu, rs = _out(), _out(), _out()
        call("scry_hip_layernorm", x.h, gamma.h, beta.h, rows, d, eps, C.byref(o), C.byref(mu),
             C.byref(rs))
        return _st(o, x.n), _st(mu, rows), _st(rs, rows)

    @staticmethod
    def layernorm_inference(x, gamma, beta, rows, d, eps=1e-5) -> Storage:
        o = _out()
        call("scry_hip_layernorm_inference", x.h, gamma.h, beta.h, rows, d, eps, C.byref(o))
        return _st(o, x.n)

    @staticmethod
    def gelu(x) -> Storage:
        o = _out()
        call("scry_hip_gelu", x.h, C.byref(o))
        return _st(o, x.n)

    @staticmethod
    def sum(x) -> float:
        out = C.c_float()
        call("scry_hip_sum", x.h, C.byref(out))
        return float(np.float32(out.value))

    @staticmethod
    def mul_elementwise(a, b) -> Storage:
        o = _out()
        call("scry_hip_mul_elementwise", a.h, b.h, C.byref(o))
        return _st(o, min(a.n, b.n))

    @staticmethod
    def concat_rows(a, b, a_rows, b_rows, cols) -> Storage:
        o = _out()
        call("scry_hip_concat_rows", a.h, b.h, a_rows, b_rows, cols, C.byref(o))
        return _st(o, a.n + b.n)

    @staticmethod
    def rope(x, rows, last_dim, pos, head_dim, theta) -> Storage:
        """MathBackend::rope on rows of last_dim values (the shape's last axis)."""
        o = _out()
        call("scry_hip_rope", x.h, rows, last_dim, pos, head_dim, theta, C.byref(o))
        return _st(o, x.n)

    @staticmethod
    def gather_columns(x, rows, total_cols, col_start, col_count) -> Storage:
        o = _out()
        call("scry_hip_gather_columns", x.h, rows, total_cols, col_start, col_count, C.byref(o))
        return _st(o, rows * col_count)

    @staticmethod
    def scatter_columns(dst, src, rows, total_cols, col_start, col_count) -> None:
        call("scry_hip_scatter_columns", dst.h, src.h, rows, total_cols, col_start, col_count)

    @staticmethod
    def gather_rows(x, total_rows, cols, row_start, row_count) -> Storage:
        o = _out()
        call("scry_hip_gather_rows", x.h, total_rows, cols, row_start, row_count, C.byref(o))
        return _st(o, row_count * cols)

    @staticmethod
    def apply_causal_mask_and_scale(scores, seq, scale, mask_value) -> None:
        call("scry_hip_apply_causal_mask_and_scale", scores.h, seq, scale, mask_value)

    @staticmethod
    def apply_batched_causal_mask_and_scale(scores, num_matrices, seq, scale, mask_value) -> None:
        call("scry_hip_apply_batched_causal_mask_and_scale", scores.h, num_matrices, seq, scale,
             mask_value)

    @staticmethod
    def split_qkv_reshape_heads(qkv, seq, n_heads, d_head):
        q, k, v = _out(), _out(), _out()
        call("scry_hip_split_qkv_reshape_heads", qkv.h, seq, n_heads, d_head, C.byref(q),
             C.byref(k), C.byref(v))
        n = seq * n_heads * d_head
        return _st(q, n), _st(k, n), _st(v, n)

    @staticmethod
    def reshape_for_heads(x, batch, seq, n_heads, d_head) -> Storage:
        o = _out()
        call("scry_hip_reshape_for_heads", x.h, batch, seq, n_heads, d_head, C.byref(o))
        return _st(o, batch * seq * n_heads * d_head)

    @staticmethod
    def reshape_from_heads(x, batch, seq, n_heads, d_head) -> Storage:
        o = _out()
        call("scry_hip_reshape_from_heads", x.h, batch, seq, n_heads, d_head, C.byref(o))
        return _st(o, batch * seq * n_heads * d_head)

    # ---- drafted tokens and the int8 KV cache (no counterpart in the reference)
    # start / lens: the context rows of each sequence (its drafted row i lies at
    # cache row len + i); parents: [n_seq, rows] or [rows], an earlier row, -1
    # (the context) or -2 (no node); None: row i follows row i - 1
    @staticmethod
    def qk_norm_rope(qkv, start, rows, n_q, n_kv, head_dim, freqs, q_weight=None, k_weight=None, eps=1e-5, q_scale=1.0,
                     parents=None) -> tuple[Storage, Storage, Storage]:
        """Per-head RMSNorm of q and k (with a weight) and RoPE at start + depth
        of the fused qkv rows [n_seq * rows, (n_q + 2 n_kv) * head_dim]."""
        st = _starts(start)
        n_seq = len(st)
        _pa, pp = _parents(parents, n_seq, rows)
        q, k, v = _out(), _out(), _out()
        call("scry_hip_qk_norm_rope", qkv.h, n_seq, rows, st.buffer_info()[0], pp, n_q, n_kv, head_dim, freqs.h,
             q_weight.h if q_weight is not None else None, k_weight.h if k_weight is not None else None, eps, q_scale,
             C.byref(q), C.byref(k), C.byref(v))
        n = n_seq * rows * head_dim
        return _st(q, n * n_q), _st(k, n * n_kv), _st(v, n * n_kv)

    @staticmethod
    def kv8_new(max_seq, n_kv, head_dim) -> KvCache8:
        o = _out()
        call("scry_hip_kv8_new", max_seq, n_kv, head_dim, C.byref(o))
        return KvCache8(o.value, max_seq, n_kv, head_dim)

    @staticmethod
    def kv8_write(caches, k, v, start, rows) -> None:
        """Quantise k, v [n_seq * rows, n_kv * head_dim] into rows start ..
        start + rows of the sequences' caches."""
        st = _starts(start)
        n_seq = len(st)
        h = _handles(caches, n_seq)
        call("scry_hip_kv8_write", h.buffer_info()[0], n_seq, st.buffer_info()[0], rows, k.h, v.h)

    @staticmethod
    def kv8_read(caches, start, rows) -> tuple[Storage, Storage]:
        """Rows start .. start + rows of the caches as f32 k and v [n_seq * rows,
        n_kv * head_dim]."""
        st = _starts(start)
        n_seq = len(st)
        h = _handles(caches, n_seq)
        k, v = _out(), _out()
        call("scry_hip_kv8_read", h.buffer_info()[0], n_seq, st.buffer_info()[0], rows, C.byref(k), C.byref(v))
        n = n_seq * rows * caches[0].n_kv * caches[0].head_dim
        return _st(k, n), _st(v, n)

    @staticmethod
    def kv8_keep(caches, start, paths) -> None:
        """The accepted paths' rows move up: row start + paths[s][i] to start + i
        (paths [n_seq, n], each ended by -1 or by n: as verify_tree returns)."""
        st = _starts(start)
        n_seq = len(st)
        p = _ints(paths, np.int64)
        if p.ndim != 2 or p.shape[0] != n_seq:
            raise ValueError(f"paths must be [{n_seq}, n]")
        h = _handles(caches, n_seq)
        call("scry_hip_kv8_keep", h.buffer_info()[0], n_seq, st.buffer_info()[0], _at(p), p.shape[1])

    @staticmethod
    def tree_attention(q, k_caches, v_caches, lens, rows, n_q, n_kv, head_dim, scale, parents=None) -> Storage:
        """Attention of drafted rows q [n_seq * rows, n_q * head_dim] over f32
        caches of rows [n_kv * head_dim]: the context and each row's ancestors."""
        st = _starts(lens)
        n_seq = len(st)
        _pa, pp = _parents(parents, n_seq, rows)
        hk, hv = _handles(k_caches, n_seq), _handles(v_caches, n_seq)
        o = _out()
        call("scry_hip_tree_attention", q.h, hk.buffer_info()[0], hv.buffer_info()[0], n_seq, st.buffer_info()[0], rows, pp,
             n_q, n_kv, head_dim, scale, C.byref(o))
        return _st(o, q.n)

    @staticmethod
    def kv8_tree_attention(q, caches, lens, rows, n_q, scale, parents=None) -> Storage:
        """tree_attention over int8 caches."""
        st = _starts(lens)
        n_seq = len(st)
        _pa, pp = _parents(parents, n_seq, rows)
        h = _handles(caches, n_seq)
        o = _out()
        call("scry_hip_kv8_tree_attention", q.h, h.buffer_info()[0], n_seq, st.buffer_info()[0], rows, pp, n_q, scale,
             C.byref(o))
        return _st(o, q.n)

    @staticmethod
    def verify_draft(p, q, tokens, u, vocab, counts=None) -> tuple[np.ndarray, np.ndarray]:
        """A drafted chain per sequence against the target's probabilities: p
        [n_seq, rows + 1, vocab], q [n_seq, rows, vocab], tokens [n_seq, rows], u
        [n_seq, rows + 1]; returns (accepted [n_seq], next token [n_seq])."""
        t = _ints(tokens, np.int64)
        if t.ndim != 2:
            raise ValueError("tokens must be [n_seq, rows]")
        n_seq, rows = t.shape
        r = np.ascontiguousarray(u, np.float64)
        if r.shape != (n_seq, rows + 1):
            raise ValueError(f"u must be [{n_seq}, {rows + 1}]")
        c = None if counts is None else _ints(counts)
        if c is not None and c.shape != (n_seq,):
            raise ValueError("one count per sequence")
        n, token = np.empty(n_seq, np.int64), np.empty(n_seq, np.int64)
        call("scry_hip_verify_draft", p.h, q.h, _at(t), None if c is None else _at(c), _at(r), n_seq,
             rows, vocab, _at(n), _at(token))
        return n, token

    @staticmethod
    def verify_tree(p, tokens, parents, u, vocab) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
        """A drafted tree per sequence: p [n_seq, rows + 1, vocab] (row 0 after
        the context, row 1 + i after node i), tokens [n_seq, rows], u [n_seq,
        rows + 1]; returns (paths [n_seq, rows], ended by -1; accepted [n_seq];
        next token [n_seq])."""
        t = _ints(tokens, np.int64)
        if t.ndim != 2:
            raise ValueError("tokens must be [n_seq, rows]")
        n_seq, rows = t.shape
        r = np.ascontiguousarray(u, np.float64)
        if r.shape != (n_seq, rows + 1):
            raise ValueError(f"u must be [{n_seq}, {rows + 1}]")
        _pa, pp = _parents(parents, n_seq, rows)
        paths = np.empty((n_seq, rows), np.int64)
        n, token = np.empty(n_seq, np.int64), np.empty(n_seq, np.int64)
        call("scry_hip_verify_tree", p.h, _at(t), pp, _at(r), n_seq, rows, vocab, _at(paths),
             _at(n), _at(token))
        return paths, n, token


def init(device: int = 0) -> None:
    HipBackend.init_gpu(device)


__all__ = ["HipBackend", "Storage", "I8Storage", "KvCache8", "init", "_lib"]
