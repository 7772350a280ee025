"""Decode attention around the BitLinear path (host mirror over libobn's C ABI).

The reference's ``Attention::forward`` (packages/rust/crates/oxbitnet/src/nn/
attention.rs:85-124) projects q/k/v with BitLinear, applies RoPE (rope.wgsl),
appends k/v to an f32 KV cache, computes scores, softmax and the weighted sum
of V (attention.wgsl, softmax.wgsl), then the o projection. Here the q/k/v
projections are one merged BitLinear whose output feeds
``rope_kv_append`` (RoPE + an fp16 cache append in one kernel) and
``attention`` (split-KV GQA attention with a combine pass); the o projection
is a BitLinear again.
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from ._lib import check, lib


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else ctypes.c_void_p(None)


def _stream(device):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


class KVCache:
    """fp16 caches [B, S_max, Hkv, head_dim] for keys and values of one layer."""

    def __init__(self, B: int, S_max: int, Hkv: int, head_dim: int = 128, device=None):
        device = device or torch.device("cuda", torch.cuda.current_device())
        self.k = torch.zeros((B, S_max, Hkv, head_dim), dtype=torch.float16, device=device)
        self.v = torch.zeros_like(self.k)
        self.B, self.S_max, self.Hkv, self.head_dim = B, S_max, Hkv, head_dim
        self.seq_len = 0


def rope_kv_append(qkv: torch.Tensor, cache: KVCache, H: int, n: int,
                   theta_base: float = 500000.0, q_out: torch.Tensor | None = None,
                   pos: int | None = None) -> torch.Tensor:
    """qkv [B*n, (H + 2*Hkv) * d] f32 of n new tokens per sequence -> rotated q
    [B*n, H*d]; k (rotated) and v stored at positions pos .. pos + n - 1
    (pos defaults to cache.seq_len)."""
    d = cache.head_dim
    q = q_out if q_out is not None else torch.empty((cache.B * n, H * d), dtype=torch.float32,
                                                     device=qkv.device)
    pos = cache.seq_len if pos is None else pos
    check(lib().obn_rope_kv_append(_ptr(qkv), cache.B, n, H, cache.Hkv, d, pos,
                                   ctypes.c_float(theta_base), _ptr(q), _ptr(cache.k),
                                   _ptr(cache.v), cache.S_max, _stream(qkv.device)))
    return q


def attention(q: torch.Tensor, cache: KVCache, H: int, n: int, seq_len: int,
              scale: float | None = None, out: torch.Tensor | None = None,
              workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal GQA attention of the n newest tokens (the cache holds seq_len
    positions per sequence): q [B*n, H*d] -> out [B*n, H*d]."""
    d = cache.head_dim
    # attention.rs: scale = 1 / sqrt(head_dim) in f32
    sc = float(np.float32(1.0) / np.sqrt(np.float32(d))) if scale is None else scale
    out = out if out is not None else torch.empty_like(q)
    need = int(lib().obn_attention_workspace_bytes(cache.B, n, H, d, seq_len))
    ws = workspace if workspace is not None and workspace.numel() >= need else \
        torch.empty(max(need, 1), dtype=torch.uint8, device=q.device)
    check(lib().obn_attention_decode(_ptr(q), _ptr(cache.k), _ptr(cache.v), cache.B, n, H,
                                     cache.Hkv, d, cache.S_max, seq_len, ctypes.c_float(sc),
                                     _ptr(out), _ptr(ws), ws.numel(), _stream(q.device)))
    return out


def attention_rope(qkv: torch.Tensor, cache: KVCache, H: int, pos: int,
                   theta_base: float = 500000.0, scale: float | None = None,
                   out: torch.Tensor | None = None,
                   workspace: torch.Tensor | None = None) -> torch.Tensor:
    """One decode token per sequence: RoPE + KV append + attention in one pass
    (bit-identical to rope_kv_append then attention with n = 1). qkv [B,
    (H + 2*Hkv) * d] unrotated -> out [B, H*d]; the token sits at position pos."""
    d = cache.head_dim
    sc = float(np.float32(1.0) / np.sqrt(np.float32(d))) if scale is None else scale
    out = out if out is not None else torch.empty((cache.B, H * d), dtype=torch.float32,
                                                  device=qkv.device)
    need = int(lib().obn_attention_workspace_bytes(cache.B, 1, H, d, pos + 1))
    ws = workspace if workspace is not None and workspace.numel() >= need else \
        torch.empty(max(need, 1), dtype=torch.uint8, device=qkv.device)
    check(lib().obn_attention_decode_rope(_ptr(qkv), _ptr(cache.k), _ptr(cache.v), cache.B, H,
                                          cache.Hkv, d, cache.S_max, pos,
                                          ctypes.c_float(theta_base), ctypes.c_float(sc),
                                          _ptr(out), _ptr(ws), ws.numel(), _stream(qkv.device)))
    cache.seq_len = max(cache.seq_len, pos + 1)
    return out


# ---- KV cache in 8 bits -------------------------------------------------------------------

Q8_BLOCK = 16  # positions that share a scale


# The current stream's handle without a Stream object, and the current device, where torch has
# these calls (its CUDA builds do): a decode step makes two such calls a layer.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                      lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _call(name: str, index: int, *args) -> None:
    """An entry point on device `index` and its current stream (the last argument)."""
    fn = getattr(lib(), name)
    if _current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        check(rc)


def _check(t, name: str, dtype, index: int, numel: int | None = None) -> None:
    """t is a contiguous tensor of this type (and size) on CUDA device `index`."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype is dtype
            and t.is_contiguous()):
        raise TypeError(f"{name} must be a contiguous {dtype} CUDA tensor")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, the others are on cuda:{index}")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name} must hold {numel} elements (got {t.numel()})")


class KVCacheQ8:
    """Caches of one layer in 8 bits: int8 codes k, v [B, S_max, Hkv, head_dim] and f32
    power-of-two scales k_scale, v_scale [B, ceil(S_max / 16), Hkv]; the row at position p
    stands for codes * scale of block p // 16. Half the bytes of KVCache."""

    def __init__(self, B: int, S_max: int, Hkv: int, head_dim: int = 128, device=None):
        device = device or torch.device("cuda", torch.cuda.current_device())
        codes = [torch.zeros((B, S_max, Hkv, head_dim), dtype=torch.int8, device=device)
                 for _ in range(2)]
        scales = [torch.zeros((B, -(-S_max // Q8_BLOCK), Hkv), dtype=torch.float32,
                              device=device) for _ in range(2)]
        self._init(codes[0], scales[0], codes[1], scales[1])

    @classmethod
    def wrap(cls, k: torch.Tensor, k_scale: torch.Tensor, v: torch.Tensor,
             v_scale: torch.Tensor) -> "KVCacheQ8":
        """A cache over existing buffers (not copied). Scales that are no powers of two count as
        they are, too; they have to be 0 or normal numbers above 0."""
        self = cls.__new__(cls)
        for t, name in ((k, "k"), (v, "v")):
            _check(t, name, torch.int8, k.get_device())
        for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            _check(t, name, torch.float32, k.get_device())
        if k.dim() != 4 or v.shape != k.shape:
            raise ValueError("k and v must be [B, S_max, Hkv, head_dim], of one shape")
        want = (k.shape[0], -(-k.shape[1] // Q8_BLOCK), k.shape[2])
        if tuple(k_scale.shape) != want or tuple(v_scale.shape) != want:
            raise ValueError(f"k_scale and v_scale must be {want}")
        self._init(k, k_scale, v, v_scale)
        return self

    def _init(self, k, k_scale, v, v_scale):
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.B, self.S_max, self.Hkv, self.head_dim = k.shape
        self.device, self.index = k.device, k.get_device()
        self.seq_len = 0

    def read(self, first: int | torch.Tensor, count: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The values of rows first .. first + count - 1 of every sequence (an int, or an
        int32 tensor [B] on the device) as f32 k, v [B, count, Hkv, head_dim]; rows outside
        the cache are zero."""
        shape = (self.B, count, self.Hkv, self.head_dim)
        k = self.k_scale.new_empty(shape)
        v = torch.empty_like(k)
        host, dev = _host_or_dev(first, self, "first")
        _call("obn_kv_read_q8", self.index, self.k.data_ptr(), self.v.data_ptr(),
              self.k_scale.data_ptr(), self.v_scale.data_ptr(), self.B, self.Hkv, self.head_dim,
              self.S_max, host, dev, count, k.data_ptr(), v.data_ptr())
        return k, v


def _host_or_dev(value, cache: KVCacheQ8, name: str) -> tuple[int, int | None]:
    """(host value, None) of an int, (0, address) of an int32 tensor [B] on the device."""
    if isinstance(value, torch.Tensor):
        _check(value, name, torch.int32, cache.index, cache.B)
        return 0, value.data_ptr()
    return _int32(value, name), None


def _int32(value, name: str) -> int:
    """An int that the C ABI takes as it is: ctypes would drop the upper bits of a larger one."""
    value = int(value)
    if not -2 ** 31 <= value < 2 ** 31:
        raise ValueError(f"{name} = {value} is no 32-bit number")
    return value


def rope_kv_append_q8(qkv: torch.Tensor, cache: KVCacheQ8, H: int, n: int,
                      theta_base: float = 500000.0, q_out: torch.Tensor | None = None,
                      pos: int | torch.Tensor | None = None) -> torch.Tensor:
    """rope_kv_append into the 8-bit cache: qkv [B*n, (H + 2*Hkv) * d] f32 -> rotated q
    [B*n, H*d]; token t of sequence b is stored at position pos + t (pos[b] + t for an int32
    tensor [B] on the device; cache.seq_len by default). Tokens whose position is outside
    the cache are not stored and get a zero q row when pos is a tensor, and are refused when
    it is an int, after which cache.seq_len is pos + n or more: calls without pos append one
    behind the other. Positions on the device leave cache.seq_len as it is."""
    B, Hkv, d = cache.B, cache.Hkv, cache.head_dim
    _check(qkv, "qkv", torch.float32, cache.index, B * n * (H + 2 * Hkv) * d)
    if q_out is None:
        q_out = qkv.new_empty((B * n, H * d))
    else:
        _check(q_out, "q_out", torch.float32, cache.index, B * n * H * d)
    host, dev = _host_or_dev(cache.seq_len if pos is None else pos, cache, "pos")
    _call("obn_rope_kv_append_q8", cache.index, qkv.data_ptr(), B, n, H, Hkv, d, host, dev,
          theta_base, q_out.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(),
          cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), cache.S_max)
    if dev is None:
        cache.seq_len = max(cache.seq_len, host + n)
    return q_out


def attention_q8_workspace(cache: KVCacheQ8, H: int, n: int) -> torch.Tensor:
    """A workspace for attention_q8 of n new tokens, at every length of the cache. One call
    at a time may use it."""
    need = int(lib().obn_attention_q8_workspace_bytes(cache.B, n, H, cache.Hkv, cache.head_dim,
                                                      cache.S_max))
    return torch.empty(max(need, 1), dtype=torch.uint8, device=cache.device)


def attention_q8(q: torch.Tensor, cache: KVCacheQ8, H: int, n: int,
                 seq_len: int | torch.Tensor, scale: float | None = None,
                 out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                 max_len: int | None = None) -> torch.Tensor:
    """Causal GQA attention of the n newest tokens over the 8-bit cache: q [B*n, H*d] -> out
    [B*n, H*d]. The sequences hold seq_len positions each (an int), or seq_len[b] (an int32
    tensor [B] on the device, at most max_len, by default the cache's S_max). Query t sees
    keys [0, seq_len - n + t]; one that sees none gives a zero row."""
    B, Hkv, d = cache.B, cache.Hkv, cache.head_dim
    size = B * n * H * d
    _check(q, "q", torch.float32, cache.index, size)
    if out is None:
        out = torch.empty_like(q)
    else:
        _check(out, "out", torch.float32, cache.index, size)
    if workspace is None:
        workspace = attention_q8_workspace(cache, H, n)
    else:
        _check(workspace, "workspace", torch.uint8, cache.index)
    host, dev = _host_or_dev(seq_len, cache, "seq_len")
    if dev is not None:
        host = cache.S_max if max_len is None else _int32(max_len, "max_len")
    _call("obn_attention_q8", cache.index, q.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(),
          cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), B, n, H, Hkv, d, cache.S_max, host,
          dev, d ** -0.5 if scale is None else scale, out.data_ptr(), workspace.data_ptr(),
          workspace.numel())
    return out
