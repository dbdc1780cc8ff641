"""Host-side mirror of the reference's operator API for the hot path, on torch CUDA tensors.

Function names and argument meaning follow ggml.h (ggml_mul_mat_idx, ggml_axpy, ggml_mul_mat,
ggml_rms_norm, ggml_norm, ggml_rope_custom, ggml_soft_max + the KQV block) so that a test written
against the reference's graph builder reads the same here.  Every function calls the CUDA library
through its C ABI; torch only provides device memory and the current stream.

Shapes use the row-major view of ggml tensors: a ggml tensor with ne = {n, T} is a torch tensor
[T, n].  Weights are `Weight` objects made by `upload_weight` (the analogue of
ggml_cuda_transform_tensor): F16 rows, or Q4_0 blocks re-laid out for aligned 128-bit loads.
"""
from __future__ import annotations

import ctypes as C
import dataclasses
import struct

import numpy as np
import torch

from . import _lib
from ._lib import PI_TYPE_F16, PI_TYPE_F32, PI_TYPE_Q4_0, check, lib

sparse_pred_threshold = 0.0        # ggml.h:2219 `extern float sparse_pred_threshold`


@dataclasses.dataclass
class Weight:
    wtype: int
    data: torch.Tensor             # uint8 device buffer: F16 rows or planar Q4_0 rows
    nrows: int
    ncols: int

    @property
    def ptr(self) -> int:
        return self.data.data_ptr()


# An operator at one token lasts a few microseconds on the device, so what these wrappers do on the host is part of its time:
# tensors that are float32 and contiguous already pass untouched, and sizes and addresses of the workspace are kept.

# (torch.cuda.current_stream() makes an object: 3.3 us a call where the number alone takes 0.2, and the nodes of an FFN 79
# instead of 64 us.  The number comes from private functions, so a torch without them gets the public one.)
_raw_stream, _raw_device = getattr(torch._C, "_cuda_getCurrentRawStream", None), getattr(torch._C, "_cuda_getDevice", None)


def _stream() -> int:
    if _raw_stream is None or _raw_device is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(_raw_device())


def _p(t):
    return None if t is None else t.data_ptr()


def _f32(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype is torch.float32 and t.is_contiguous() else t.contiguous().float()


def _rows(t: torch.Tensor, T: int, n: int) -> torch.Tensor:
    """t as contiguous float32 [T, n] (either may be -1)"""
    t = _f32(t)
    if t.dim() == 2 and (T < 0 or t.shape[0] == T) and (n < 0 or t.shape[1] == n):
        return t
    return t.reshape(T, n)


class Workspace:
    """Scratch for the operators below, grown on demand (the C ABI itself never allocates)."""

    def __init__(self):
        self.buf = None
        self.at = self.size = 0
        self.need: dict = {}                 # (ncols, nrows, T) -> bytes
        self.asked = None                    # where the last operator's status word is: (address, the tensor that holds it); None: it has none

    def get(self, ncols: int, nrows: int, T: int):
        need = self.need.get((ncols, nrows, T))
        if need is None:
            if len(self.need) > 1024:
                self.need.clear()
            need = self.need[(ncols, nrows, T)] = lib.pi_workspace_bytes(ncols, nrows, T)
        if self.buf is None or self.buf.numel() < need:
            self.buf = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
            off = (-self.buf.data_ptr()) % 256
            self.at, self.size = self.buf.data_ptr() + off, self.buf.numel() - off
        self.asked = self.at, self.buf
        return self.at, self.size


_ws = Workspace()


def last_op_status() -> int:
    """Status of the last operator issued through this module (pi_op_status): 0, or 5 (a bounded device-side wait ran out)."""
    if _ws.asked is None:
        return 0
    return int(lib.pi_op_status(_ws.asked[0], _stream()))


def upload_weight(host: np.ndarray, wtype: int, nrows: int, ncols: int) -> Weight:
    """host: float16 [nrows, ncols], or uint8 ggml Q4_0 blocks [nrows, ncols/32*18]."""
    if wtype == PI_TYPE_F16:
        assert host.dtype == np.float16 and host.shape == (nrows, ncols)
        dev = torch.from_numpy(np.ascontiguousarray(host).view(np.uint8).reshape(-1)).cuda()
        return Weight(wtype, dev, nrows, ncols)
    raw = torch.from_numpy(np.ascontiguousarray(host, np.uint8).reshape(-1)).cuda()
    assert raw.numel() == nrows * (ncols // 32) * 18
    dev = torch.empty_like(raw)
    check(lib.pi_q4_0_repack(raw.data_ptr(), dev.data_ptr(), nrows, ncols, _stream()))
    return Weight(wtype, dev, nrows, ncols)


def quantize_q4_0(x: torch.Tensor) -> torch.Tensor:
    """F32 [rows, cols] on device -> ggml Q4_0 block bytes (uint8 [rows*cols/32*18])."""
    x = x.contiguous().float()
    out = torch.empty(x.numel() // 32 * 18, dtype=torch.uint8, device=x.device)
    check(lib.pi_quantize_q4_0(x.data_ptr(), out.data_ptr(), x.shape[0], x.shape[1], _stream()))
    return out


def quantize_q8_0(x: torch.Tensor) -> torch.Tensor:
    x = x.contiguous().float()
    out = torch.empty(x.numel() // 32 * 34, dtype=torch.uint8, device=x.device)
    check(lib.pi_quantize_q8_0(x.data_ptr(), out.data_ptr(), x.shape[0], x.shape[1], _stream()))
    return out


def dequantize(w: Weight) -> torch.Tensor:
    if w.wtype == PI_TYPE_F16:
        return w.data.view(torch.float16).reshape(w.nrows, w.ncols).float()
    out = torch.empty(w.nrows, w.ncols, dtype=torch.float32, device="cuda")
    check(lib.pi_dequantize_q4_0(w.ptr, out.data_ptr(), w.nrows, w.ncols, _stream()))
    return out


def ggml_mul_mat(a: Weight, b: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """ggml_mul_mat(ctx, a, b): a [nrows, ncols] weights, b F32 [T, ncols] -> F32 [T, nrows]."""
    b = _rows(b, -1, a.ncols)
    T = b.shape[0]
    dst = torch.empty(T, a.nrows, dtype=torch.float32, device="cuda")
    ws, wsn = _ws.get(a.ncols, a.nrows, T)
    check(lib.pi_mul_mat(a.wtype, a.ptr, a.nrows, a.ncols, b.data_ptr(), T, _p(bias), dst.data_ptr(), ws, wsn, _stream()))
    return dst


def ggml_mul_mat_idx(a: Weight, b: torch.Tensor, sparse_idx: torch.Tensor, gpu_bucket: torch.Tensor | None = None,
                     result_ne0: int | None = None) -> torch.Tensor:
    """ggml_mul_mat_idx / ggml_mul_mat_idx_upscale (ggml.h:1094-1106).

    a: rows of up / gate held on this device; b: F32 [T, ncols]; sparse_idx: F32 [T, F] predictor logits by
    global neuron id; gpu_bucket: int32 [a.nrows] global ids of a's rows (None: a holds all F rows);
    result_ne0: F when a bucket is given.  Returns F32 [T, F]."""
    b = _rows(b, -1, a.ncols)
    T = b.shape[0]
    sparse_idx = _rows(sparse_idx, T, -1)
    F = result_ne0 if gpu_bucket is not None else a.nrows
    assert F is not None and sparse_idx.shape[1] >= F
    dst = torch.empty(T, F, dtype=torch.float32, device="cuda")
    ws, wsn = _ws.get(a.ncols, max(a.nrows, F), T)
    check(lib.pi_mul_mat_idx(a.wtype, a.ptr, a.nrows, a.ncols, b.data_ptr(), T, sparse_idx.data_ptr(),
                             sparse_idx.shape[1], _p(gpu_bucket), sparse_pred_threshold, dst.data_ptr(), F,
                             ws, wsn, _stream()))
    return dst


def ggml_axpy(a: Weight, b: torch.Tensor, sparse_idx: torch.Tensor, hybrid_aux: torch.Tensor | None = None) -> torch.Tensor:
    """ggml_axpy (ggml.h:1107-1112): a = rows of ffn_down_t on this device, b = F32 [T, F] hidden activations,
    hybrid_aux = gpu_bucket (int32 [a.nrows]) or None.  Returns F32 [T, ncols]."""
    T = b.shape[0] if b.dim() == 2 else 1
    b = _rows(b, T, -1)
    sparse_idx = _rows(sparse_idx, T, -1)
    dst = torch.empty(T, a.ncols, dtype=torch.float32, device="cuda")
    ws, wsn = _ws.get(a.ncols, max(a.nrows, b.shape[1]), T)
    check(lib.pi_axpy(a.wtype, a.ptr, a.nrows, a.ncols, b.data_ptr(), T, b.shape[1], sparse_idx.data_ptr(),
                      sparse_idx.shape[1], _p(hybrid_aux), sparse_pred_threshold, dst.data_ptr(), ws, wsn, _stream()))
    return dst


def sparse_ffn(up: Weight, gate: Weight | None, down_t: Weight, x: torch.Tensor, sparse_idx: torch.Tensor,
               gpu_bucket: torch.Tensor | None = None, up_bias: torch.Tensor | None = None) -> torch.Tensor:
    """llm_build_ffn_sparse (llama.cpp:4652-4757) after the predictor, as one call: the two ggml_mul_mat_idx nodes, the
    relu / mul / bias nodes and ggml_axpy.  x F32 [T, d], sparse_idx F32 [T, F] -> F32 [T, d]."""
    x = _rows(x, -1, up.ncols)
    T = x.shape[0]
    sparse_idx = _rows(sparse_idx, T, -1)
    F = sparse_idx.shape[1]
    dst = torch.empty(T, up.ncols, dtype=torch.float32, device="cuda")
    ws, wsn = _ws.get(up.ncols, max(up.nrows, F), T)
    check(lib.pi_sparse_ffn(up.wtype, up.ptr, gate.ptr if gate is not None else None, down_t.ptr, up.nrows, up.ncols,
                            x.data_ptr(), T, sparse_idx.data_ptr(), F, _p(gpu_bucket), sparse_pred_threshold, _p(up_bias),
                            dst.data_ptr(), ws, wsn, _stream()))
    return dst


def predictor(fc1: Weight, fc2: Weight, p: torch.Tensor) -> torch.Tensor:
    """idx = mul_mat(fc2, relu(mul_mat(fc1, p))) (llama.cpp:4688-4695); p F32 [T, d] -> F32 [T, F]."""
    p = _rows(p, -1, fc1.ncols)
    T = p.shape[0]
    idx = torch.empty(T, fc2.nrows, dtype=torch.float32, device="cuda")
    ws, wsn = _ws.get(max(fc1.ncols, fc2.ncols), max(fc1.nrows, fc2.nrows), T)
    check(lib.pi_predictor(fc1.ptr, fc2.ptr, fc1.ncols, fc1.nrows, fc2.nrows, p.data_ptr(), T, idx.data_ptr(), ws, wsn, _stream()))
    return idx


def active_list(sparse_idx: torch.Tensor):
    """Sorted ids of neurons whose logit >= threshold for at least one token, and their count (device tensors)."""
    sparse_idx = sparse_idx.contiguous().float()
    T, F = (sparse_idx.shape[0], sparse_idx.shape[1]) if sparse_idx.dim() == 2 else (1, sparse_idx.numel())
    lst = torch.empty(F, dtype=torch.int32, device="cuda")
    cnt = torch.zeros(1, dtype=torch.int32, device="cuda")
    ws, wsn = _ws.get(F, F, T)
    check(lib.pi_active_list(sparse_idx.data_ptr(), F, T, F, sparse_pred_threshold, lst.data_ptr(), cnt.data_ptr(), ws, wsn, _stream()))
    return lst, cnt


def _norm(x, rms, eps, w, b):
    x = x.contiguous().float()
    x2 = x.reshape(-1, x.shape[-1])
    y = torch.empty_like(x2)
    check(lib.pi_norm(x2.data_ptr(), x2.shape[0], x2.shape[1], rms, eps, _p(w), _p(b), y.data_ptr(), _stream()))
    return y.reshape(x.shape)


def ggml_rms_norm(x, eps, w=None, b=None):
    """ggml_rms_norm followed by llm_build_norm's optional weight and bias."""
    return _norm(x, 1, eps, w, b)


def ggml_norm(x, eps, w=None, b=None):
    return _norm(x, 0, eps, w, b)


def rope_table(n_pos: int, head_dim: int, freq_base: float) -> torch.Tensor:
    host = np.empty((n_pos, head_dim // 2, 2), np.float32)
    lib.pi_rope_table_host(host.ctypes.data, n_pos, head_dim, freq_base)
    return torch.from_numpy(host).cuda()


def ggml_rope_custom(x: torch.Tensor, pos: torch.Tensor, n_dims: int, mode: int, table: torch.Tensor) -> torch.Tensor:
    """x F32 [T, n_heads, n_dims]; pos int32 [T]; mode 0 or 2 (neox)."""
    y = x.contiguous().float().clone()
    T, n_heads = y.shape[0], y.shape[1]
    check(lib.pi_rope(y.data_ptr(), T, n_heads, n_dims, pos.data_ptr(), table.data_ptr(), 1 if mode & 2 else 0, _stream()))
    return y


def attention_decode(q, k, v, k_cache, v_cache, pos, n_head, n_head_kv, seq=None):
    """KV store + KQV block for one new token per sequence.  q [T, n_head*hd], k/v [T, n_head_kv*hd] (RoPE'd),
    caches float16 [n_seq, n_ctx, n_head_kv*hd] updated in place.  Returns F32 [T, n_head*hd]."""
    T = q.shape[0]
    hd = q.shape[1] // n_head
    out = torch.empty(T, n_head * hd, dtype=torch.float32, device="cuda")
    check(lib.pi_attention_decode(q.data_ptr(), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                  _p(seq), pos.data_ptr(), T, n_head, n_head_kv, hd, k_cache.shape[1], out.data_ptr(), _stream()))
    return out


# ---- a long context: scaled rotary positions, a KV cache in 8 bits, its attention and eviction.
# Rows are float32 or float16 and may be columns of a wider matrix (q, k and v as one projection leaves them); results are new tensors.
# Scratch and results come from torch's allocator at every call, so calls on several streams and captured graphs share none.
# (Every attribute of a tensor costs 0.1 to 0.3 us: it is asked for once.  The two C structures are packed bytes: 0.5 us each, ctypes' own 1.5.)

_ROW_TYPES = {torch.float32: PI_TYPE_F32, torch.float16: PI_TYPE_F16}
_KV_Q8 = struct.Struct("@4P5i4x")          # pi_kv_q8
_KV_BATCH = struct.Struct("@3P3i4x")       # pi_kv_batch
assert _KV_Q8.size == C.sizeof(_lib.KvQ8) and _KV_BATCH.size == C.sizeof(_lib.KvBatch)


def _here(*tensors):
    device = torch.cuda.current_device() if _raw_device is None else _raw_device()
    for t in tensors:
        if t is not None and t.get_device() != device:
            raise ValueError(f"a tensor is on {t.device}, the current device is cuda:{device}")


def _row_matrix(t: torch.Tensor, what: str, width: int = 0):
    """t [T, n] (or [T, heads, head_dim]) as rows that the kernels take, 16-byte aligned and a row's values side by side (a copy where it is not):
    (tensor, address, rows, values of a row, values between rows, type)"""
    shape = t.shape
    if len(shape) == 3:
        t = t.flatten(1)
        shape = t.shape
    if len(shape) != 2:
        raise ValueError(f"{what} must have 2 or 3 dimensions: rows of heads")
    T, n = shape
    xtype = _ROW_TYPES.get(t.dtype)
    if xtype is None:
        raise ValueError(f"{what} is {t.dtype}: float32 or float16 is needed")
    if width and n != width:
        raise ValueError(f"{what} is [{T}, {n}]: rows of {width} values are needed")
    step, side = t.stride()
    at = t.data_ptr()
    if T <= 1:
        step = n
    if side != 1 or at % 16 or step < n or step * (2 if xtype == PI_TYPE_F16 else 4) % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        step, at = n, t.data_ptr()
    return t, at, T, n, step, xtype


def _ints(t: torch.Tensor, n: int, what: str) -> int:
    if t.dtype is not torch.int32 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 tensor of {n}")
    return t.data_ptr()


class RopeFreqs:
    """freqs: float64 [n_rot / 2] on the device, the angle per position of each pair; mscale: factor of the rotated values"""

    __slots__ = ("freqs", "mscale")

    def __init__(self, freqs: torch.Tensor, mscale: float = 1.0):
        if freqs.dtype is not torch.float64 or not freqs.is_contiguous():
            raise ValueError("frequencies must be contiguous float64")
        self.freqs, self.mscale = freqs, mscale


def rope_freqs(n_rot: int, freq_base: float = 10000.0, freq_scale: float = 1.0, ext_factor: float = 0.0, attn_factor: float = 1.0,
               beta_fast: float = 32.0, beta_slow: float = 1.0, n_orig_ctx: int = 0, freq_factors=None) -> RopeFreqs:
    """The parameters of ggml_rope_custom (ggml.h:1266-1283) as frequencies: made once, like rope_table."""
    host, mscale = np.empty(max(0, n_rot) // 2, np.float64), C.c_float(1.0)
    factors = None if freq_factors is None else np.ascontiguousarray(freq_factors, np.float32)
    if factors is not None and factors.shape != host.shape:
        raise ValueError(f"freq_factors must be {host.shape[0]} values")
    check(lib.pi_rope_freqs_host(host.ctypes.data, C.addressof(mscale), n_rot, freq_base, freq_scale, ext_factor, attn_factor, beta_fast, beta_slow,
                                 n_orig_ctx, None if factors is None else factors.ctypes.data))
    return RopeFreqs(torch.from_numpy(host).cuda(), mscale.value)


def rope_ext(q: torch.Tensor, k: torch.Tensor | None, pos: torch.Tensor, freqs: RopeFreqs, head_dim: int, mode: int = 0, inplace: bool = False):
    """Queries [T, n_head * head_dim] and keys [T, n_head_kv * head_dim] rotated to pos int32 [T]; mode 0 (pairs (2i, 2i+1)) or 2 (neox).  The first
    2 * len(freqs) dimensions of each head turn.  Returns (q, k): new tensors of rows (two dimensions, also for [T, heads, head_dim]), or the same ones with inplace."""
    xq, q_at, T, nq, q_step, xtype = _row_matrix(q, "q")
    f = freqs.freqs
    if nq % head_dim:
        raise ValueError(f"q has rows of {nq} values: heads of {head_dim} are needed")
    if inplace:
        yq, yq_at, yq_step = q, q_at, q_step
        if q_at != q.data_ptr():
            raise ValueError("in place needs rows that are 16-byte aligned")
    else:
        yq, yq_step = torch.empty_like(xq), nq                       # (contiguous: xq's rows are, or lie apart)
        yq_at = yq.data_ptr()
    if k is None:
        _here(xq, pos, f)
        check(lib.pi_rope_ext(xtype, q_at, q_step, nq // head_dim, yq_at, yq_step, None, 0, 0, None, 0, T, head_dim, 2 * f.numel(), 1 if mode & 2 else 0,
                              _ints(pos, T, "pos"), f.data_ptr(), freqs.mscale, _stream()))
        return yq, None
    xk, k_at, Tk, nk, k_step, ktype = _row_matrix(k, "k")
    if Tk != T or ktype != xtype or nk % head_dim:
        raise ValueError(f"q and k must be of one type, {T} rows of heads of {head_dim}")
    if inplace:
        yk, yk_at, yk_step = k, k_at, k_step
        if k_at != k.data_ptr():
            raise ValueError("in place needs rows that are 16-byte aligned")
    else:
        yk, yk_step = torch.empty_like(xk), nk
        yk_at = yk.data_ptr()
    _here(xq, xk, pos, f)
    check(lib.pi_rope_ext(xtype, q_at, q_step, nq // head_dim, yq_at, yq_step, k_at, k_step, nk // head_dim, yk_at, yk_step, T, head_dim, 2 * f.numel(),
                          1 if mode & 2 else 0, _ints(pos, T, "pos"), f.data_ptr(), freqs.mscale, _stream()))
    return yq, yk


class KvCacheQ8:
    """A KV cache in 8 bits: codes int8 [n_seq, n_head_kv, n_ctx, head_dim], scales float32 [n_seq, n_head_kv, n_ctx / block]."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "n_seq", "n_head_kv", "n_ctx", "head_dim", "block", "c")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        shape, blocks = k.shape, k_scale.shape
        if k.dtype is not torch.int8 or v.dtype is not torch.int8 or k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32:
            raise ValueError("codes are int8, scales float32")
        if len(shape) != 4 or len(blocks) != 3 or v.shape != shape or v_scale.shape != blocks or blocks[:2] != shape[:2] or not blocks[2] or shape[2] % blocks[2]:
            raise ValueError("codes [n_seq, n_head_kv, n_ctx, head_dim] and scales [n_seq, n_head_kv, n_ctx / block] do not fit each other")
        if not (k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
            raise ValueError("the caches must be contiguous")
        _here(k, v, k_scale, v_scale)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        n_seq, n_head_kv, n_ctx, head_dim = shape
        self.n_seq, self.n_head_kv, self.n_ctx, self.head_dim, self.block = n_seq, n_head_kv, n_ctx, head_dim, n_ctx // blocks[2]
        self.c = _KV_Q8.pack(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), n_seq, n_head_kv, n_ctx, head_dim, self.block)

    @classmethod
    def empty(cls, n_seq: int, n_ctx: int, n_head_kv: int, head_dim: int, block: int = 64) -> "KvCacheQ8":
        if block <= 0 or n_ctx <= 0 or n_ctx % block:
            raise ValueError(f"n_ctx={n_ctx} must be a multiple of block={block}")
        codes = [torch.zeros(n_seq, n_head_kv, n_ctx, head_dim, dtype=torch.int8, device="cuda") for _ in range(2)]
        return cls(*codes, *(torch.zeros(n_seq, n_head_kv, n_ctx // block, device="cuda") for _ in range(2)))


def _batch(q_start, pos0, seq, T, max_new) -> bytes:
    n = pos0.numel()
    return _KV_BATCH.pack(_ints(q_start, n + 1, "q_start"), 0 if seq is None else _ints(seq, n, "seq"), _ints(pos0, n, "pos0"), n, T,
                          T if max_new is None else max_new)


def kv_store_q8(cache: KvCacheQ8, k: torch.Tensor, v: torch.Tensor, q_start: torch.Tensor, pos0: torch.Tensor, seq: torch.Tensor | None = None,
                max_new: int | None = None) -> None:
    """k, v [T, n_head_kv * head_dim] into the cache: rows q_start[i] .. q_start[i + 1] to the slots pos0[i] and on of sequence seq[i] (None: i); at
    most max_new rows of an entry (None: T)."""
    width = cache.n_head_kv * cache.head_dim
    k, k_at, T, _, k_step, xtype = _row_matrix(k, "k", width)
    v, v_at, Tv, _, v_step, vtype = _row_matrix(v, "v", width)
    if Tv != T or vtype != xtype:
        raise ValueError("k and v must have the same rows and type")
    _here(cache.k, k, v, q_start, pos0, seq)
    check(lib.pi_kv_store_q8(cache.c, _batch(q_start, pos0, seq, T, max_new), xtype, k_at, k_step, v_at, v_step, _stream()))


def kv_load_q8(cache: KvCacheQ8, q_start: torch.Tensor, pos0: torch.Tensor, T: int, seq: torch.Tensor | None = None, max_new: int | None = None,
               dtype: torch.dtype = torch.float32):
    """The values of the slots that kv_store_q8 with the same batch writes: k, v [T, n_head_kv * head_dim] (rows of no entry hold anything)."""
    width, xtype = cache.n_head_kv * cache.head_dim, _ROW_TYPES.get(dtype)
    if xtype is None:
        raise ValueError("values are read as float32 or float16")
    k = cache.k_scale.new_empty(T, width) if dtype is torch.float32 else cache.k_scale.new_empty(T, width, dtype=dtype)
    v = torch.empty_like(k)
    _here(cache.k, q_start, pos0, seq)
    check(lib.pi_kv_load_q8(cache.c, _batch(q_start, pos0, seq, T, max_new), xtype, k.data_ptr(), width, v.data_ptr(), width, _stream()))
    return k, v


def _slot_weights(w: torch.Tensor | None, cache: KvCacheQ8):
    if w is None:
        return None
    if w.dtype is not torch.float32 or w.shape != (cache.n_seq, cache.n_head_kv, cache.n_ctx) or not w.is_contiguous():
        raise ValueError("weights are contiguous float32 [n_seq, n_head_kv, n_ctx]")
    return w.data_ptr()


def attention_q8(cache: KvCacheQ8, q: torch.Tensor, q_start: torch.Tensor, pos0: torch.Tensor, seq: torch.Tensor | None = None, max_new: int | None = None,
                 max_kv: int | None = None, scale: float | None = None, weights_in: torch.Tensor | None = None, weights_out: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """The KQV block over the 8-bit cache, the batch's own keys and values stored before: q [T, n_head * head_dim] (or [T, n_head, head_dim]) -> rows of q's type.  Token t
    of entry i sees the slots up to pos0[i] + t.  max_kv: slots that the longest sequence sees (None: all).  weights_out float32 [n_seq,
    n_head_kv, n_ctx] takes each seen slot's probabilities, plus weights_in for slots before pos0.  Rows of no entry are left as `out` has them."""
    hd = cache.head_dim
    q, q_at, T, n, q_step, xtype = _row_matrix(q, "q")
    if n % hd:
        raise ValueError(f"q has rows of {n} values: heads of {hd} are needed")
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != (T, n) or out.dtype is not q.dtype or not out.is_contiguous():
        raise ValueError("out must be contiguous, of q's shape and type")
    w_in, w_out = _slot_weights(weights_in, cache), _slot_weights(weights_out, cache)
    _here(cache.k, q, out, q_start, pos0, seq, weights_in, weights_out)
    b, most = _batch(q_start, pos0, seq, T, max_new), cache.n_ctx if max_kv is None else max_kv
    need = lib.pi_attention_q8_workspace_bytes(cache.c, b, n // hd, most, 0 if w_out is None else 1)
    _ws.asked = ws_at = None                                          # (the former call's scratch goes back first)
    if need:
        ws = cache.k.new_empty(need)
        ws_at = ws.data_ptr()
        if (hd == 64 or hd == 128) and min(T, T if max_new is None else max_new) * (n // hd // cache.n_head_kv) >= 64:
            _ws.asked = ws_at, ws                                     # (the calls with bounded waits; kept until the next operator, for last_op_status)
    check(lib.pi_attention_q8(cache.c, b, xtype, q_at, q_step, n // hd, most, hd ** -0.5 if scale is None else scale, out.data_ptr(), n, w_in, w_out, ws_at, need, _stream()))
    return out


def kv_evict_q8(cache: KvCacheQ8, weights: torch.Tensor, lens: torch.Tensor, keep: int, n_sink: int = 4, n_recent: int = 0, seq: torch.Tensor | None = None,
                weights_out: torch.Tensor | None = None) -> torch.Tensor:
    """Sequences of lens[i] slots cut to `keep` by their accumulated weights (float32 [n_seq, n_head_kv, n_ctx], as attention_q8 leaves them): the first
    n_sink slots, the last n_recent and the heaviest others stay, for every KV head its own.  Returns the slot that each kept row came from,
    int32 [n, n_head_kv, keep] (-1: none); weights_out (may be `weights`) takes the weights in the new order.
    Kept slots behind `keep` move into the places of evicted ones below it.  So the last n_recent slots are the newest tokens only if every eviction takes n_recent
    slots or more (lens[i] - keep >= n_recent): let a sequence grow to keep + n_recent before it is cut.  Cut at every token, it has no recent window."""
    n = lens.numel()
    w, w_out = _slot_weights(weights, cache), _slot_weights(weights_out, cache)
    _here(cache.k, weights, weights_out, lens, seq)
    kept = lens.new_empty(n, cache.n_head_kv, max(0, keep))
    check(lib.pi_kv_evict_q8(cache.c, _ints(lens, n, "lens"), None if seq is None else _ints(seq, n, "seq"), n, keep, n_sink, n_recent, w, w_out,
                             kept.data_ptr(), _stream()))
    return kept
