"""Paged key/value cache: appending new tokens and causal attention over the pages, for prompts and single tokens.

Host-side mirror of the f2k_kv_* part of include/f2k_attn.h, in the manner of the attention modules: an object is
configured once, calls return False and `last_error()` explains, tensors are CUDA tensors of the caller. A tensor of
the wrong type, shape or device raises TypeError.

    kv = PagedKV(PagedKV.Config(32, 8, 128, page_size=16, n_pages=4096, rot_dim=128), k_pages, v_pages)
    batch = PagedBatch(kv_lens, page_table, cu_seqlens, max_new=512)      # lengths with the new tokens
    ws = torch.empty(kv.workspace_size_bytes(batch), dtype=torch.uint8, device="cuda")
    kv.append(q, k, v, (gamma_q, gamma_k), (cos, sin), 1e-6, q, batch) and kv.attend(q, o, batch, ws)
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import KvBatch, KvConfig, lib
from ._stream import stream_handle

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float8_e4m3fn: 2}


# struct f2k_kv_append_args, f2k_kv_attend_args: written whole by one call. (As 14 arguments of the C function, each
# converted by ctypes, they cost the host 2 us more.)
_APPEND = struct.Struct("8Q4qif")
_ATTEND = struct.Struct("3Q2q2Q")


def _p(t):
    return 0 if t is None else t.data_ptr()


def _strides(pages):
    """Page, head and token stride; of a dimension of one element, whose stride says nothing, that of a dense array."""
    dense = pages.shape[1] * pages.shape[2] * pages.shape[3], pages.shape[2] * pages.shape[3], pages.shape[3]
    return [s if n > 1 else d for n, s, d in zip(pages.shape, pages.stride(), dense)]


class PagedBatch:
    """The sequences of a call. kv_lens int32 [n]: lengths with the new tokens. page_table int32 [n, width], rows may be
    strided. cu_seqlens int32 [n + 1]: rows of the new tokens; None: one each. max_new: the most new tokens that a
    sequence has. The tensors are read by the kernels when they run, so a captured call follows what is written to them."""

    def __init__(self, kv_lens, page_table, cu_seqlens=None, max_new: int = 1):
        n = kv_lens.shape[0]
        for t, dims in ((kv_lens, 1), (page_table, 2), (cu_seqlens, 1)):
            if t is not None and (t.dtype is not torch.int32 or t.dim() != dims or (t.shape[-1] > 1 and t.stride(-1) != 1)
                                  or t.device != kv_lens.device):
                raise TypeError("lengths and page table must be int32 on one device, rows contiguous")
        if n > 1 and page_table.stride(0) < page_table.shape[1]:      # an expanded row: 0 would mean dense
            raise TypeError("the rows of page_table must not overlap")
        if page_table.shape[0] != n or (cu_seqlens is not None and cu_seqlens.shape[0] != n + 1):
            raise TypeError("kv_lens [n], page_table [n, width] and cu_seqlens [n + 1] belong together")
        if cu_seqlens is None and max_new != 1:
            raise TypeError("without cu_seqlens every sequence has one new token")
        self.kv_lens, self.page_table, self.cu_seqlens, self.max_new = kv_lens, page_table, cu_seqlens, max_new
        self.index = kv_lens.get_device()
        self._c = KvBatch(n, 0, max_new, page_table.shape[1], page_table.stride(0) if n > 1 else 0, _p(cu_seqlens), _p(kv_lens),
                          _p(page_table))
        self._ref = C.byref(self._c)

    def _with(self, n_tokens):
        self._c.n_tokens = n_tokens
        return self._ref


class PagedKV:
    """One layer's cache. k_pages, v_pages: [n_pages, n_kv_heads, page_size, head_dim] tensors or views in that order of
    dimensions, of Config.dtype or float8_e4m3fn; k_scale, v_scale: fp32 [n_kv_heads], e4m3 only."""

    @dataclass
    class Config:
        n_heads: int = 0
        n_kv_heads: int = 0
        head_dim: int = 0
        page_size: int = 0
        n_pages: int = 0
        rot_dim: int = 0            # 0: no rotation
        interleaved: bool = False   # pairs (2i, 2i+1) instead of (i, i + rot_dim/2)
        window: int = 0             # 0: no window
        scale: float = 0.0          # 0: 1/sqrt(head_dim)
        dtype: torch.dtype = torch.bfloat16

    def __init__(self, cfg: "PagedKV.Config", k_pages, v_pages, k_scale=None, v_scale=None):
        self._h = C.c_void_p()
        self.cfg = cfg
        shape = (cfg.n_pages, cfg.n_kv_heads, cfg.page_size, cfg.head_dim)
        if cfg.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError("dtype must be bfloat16 or float16")
        for t in (k_pages, v_pages):
            if tuple(t.shape) != shape or t.dtype not in _TYPES or t.dtype != k_pages.dtype or t.device != k_pages.device \
                    or t.stride(3) != 1:
                raise TypeError(f"pages must be {list(shape)}, both of one type and device, rows contiguous")
            if any(n > 1 and s <= 0 for n, s in zip(shape, t.stride())):
                raise TypeError("pages must not be expanded")
        for t in (k_scale, v_scale):
            if t is not None and (t.dtype is not torch.float32 or tuple(t.shape) != (cfg.n_kv_heads,) or not t.is_contiguous()
                                  or t.device != k_pages.device):
                raise TypeError("scales must be contiguous float32 [n_kv_heads] on the pages' device")
        self.k_pages, self.v_pages, self.k_scale, self.v_scale = k_pages, v_pages, k_scale, v_scale
        self.device, self._index = k_pages.device, k_pages.get_device()
        self._args = bytearray(max(_APPEND.size, _ATTEND.size))       # a handle is used from one thread at a time
        self._args_at = C.addressof(C.c_char.from_buffer(self._args))
        self._dtype, self._heads, self._kv_heads, self._dim, self._half = cfg.dtype, cfg.n_heads, cfg.n_kv_heads, cfg.head_dim, cfg.rot_dim // 2
        self._gain = (cfg.head_dim,)
        c = KvConfig(cfg.n_heads, cfg.n_kv_heads, cfg.head_dim, cfg.page_size, cfg.n_pages, _TYPES[cfg.dtype],
                     _TYPES[k_pages.dtype], cfg.rot_dim, int(cfg.interleaved), cfg.window, cfg.scale, _p(k_pages), _p(v_pages),
                     *_strides(k_pages), *_strides(v_pages), _p(k_scale), _p(v_scale))
        self._rc = lib.f2k_kv_create(C.byref(c), C.byref(self._h))

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h and lib is not None:
            lib.f2k_kv_destroy(h)

    def ok(self) -> bool:
        return self._rc == _lib.F2K_OK

    def last_error(self) -> str:
        return lib.f2k_kv_last_error(self._h).decode() if self._h else "no handle"

    def device_status(self) -> int:
        """Synchronises; 0 means every kernel of this cache ran clean."""
        st = C.c_int(0)
        lib.f2k_kv_device_status(self._h, C.byref(st))
        return st.value

    def set_wait_limits(self, in_cta_clk: int = 0) -> bool:
        return lib.f2k_kv_set_wait_limits(self._h, in_cta_clk) == _lib.F2K_OK

    def workspace_size_bytes(self, batch: PagedBatch) -> int:
        return int(lib.f2k_kv_workspace_bytes(self._h, batch._ref)) if self.ok() else 0

    # The checks are most of what a call of a few tokens costs the host (8 appended tokens 9.9 us a call when every tensor's
    # strides and device object were looked at), so the plain case asks little.
    def _stride(self, t, wanted):
        """Token stride of a tensor of the layer, `wanted` [rows, heads, head_dim]; 0: dense. A dense one may have its rows in several
        dimensions, and a token's heads in one."""
        if t.dtype is not self._dtype or t.get_device() != self._index:
            raise TypeError(f"expected {self._dtype} on {self.device}")
        shape = t.shape
        if t.is_contiguous() and (shape == wanted or t.numel() == math.prod(wanted)
                                  and (shape[-1] == wanted[1] * wanted[2] or shape[-2:] == wanted[1:])):
            return 0
        s, (rows, heads, dim) = t.stride(), wanted
        if shape != wanted or s[2] != 1 or (heads > 1 and s[1] != dim) or (rows > 1 and s[0] < heads * dim):
            raise TypeError(f"expected {list(wanted)}, a token's heads dense, rows apart")
        return s[0] if rows > 1 else 0

    def _vector(self, t, dtype, shape, what):
        """Address of a dense tensor of this shape, or of another with as many elements whose rows, if it has any, are as long."""
        if t.dtype is not dtype or t.get_device() != self._index or not t.is_contiguous() \
                or (t.shape != shape and (t.numel() != math.prod(shape) or (t.dim() > 1 and t.shape[-1] != shape[-1]))):
            raise TypeError(f"{what} must be contiguous {dtype} {list(shape)} on {self.device}")
        return t.data_ptr()

    def append(self, Q, K, V, gammas, tables, eps, Q_out, batch: PagedBatch, stream=None) -> bool:
        """K and V of the batch's new tokens into the cache, Q to Q_out (which may be Q), both normalised and rotated on the
        way. gammas = (gamma_q, gamma_k), [head_dim] of Config.dtype, or (None, None); tables = (cos, sin), fp32
        [positions, rot_dim / 2], or (None, None) with rot_dim 0."""
        if self._rc:
            return False
        n, stride = Q.shape[0], self._stride
        q_shape, kv_shape = (n, self._heads, self._dim), (n, self._kv_heads, self._dim)
        gamma_q, gamma_k = gammas
        cos, sin = tables
        positions, table = 0, (0, self._half)
        if cos is not None and self._half:
            positions = cos.shape[0]
            table = positions, self._half
            cos = self._vector(cos, torch.float32, table, "tables")
        if sin is not None and self._half:
            sin = self._vector(sin, torch.float32, table, "tables")
        if gamma_q is not None:
            gamma_q = self._vector(gamma_q, self._dtype, self._gain, "gains")
        if gamma_k is not None:
            gamma_k = self._vector(gamma_k, self._dtype, self._gain, "gains")
        if batch.index != self._index:
            raise TypeError("the batch lies on another device than the cache")
        _APPEND.pack_into(self._args, 0, Q.data_ptr(), K.data_ptr(), V.data_ptr(), gamma_q or 0, gamma_k or 0,
                          cos if self._half and cos else 0, sin if self._half and sin else 0, Q_out.data_ptr(),
                          stride(Q, q_shape), stride(K, kv_shape), stride(V, kv_shape), stride(Q_out, q_shape),
                          positions, eps)
        return lib.f2k_kv_append(self._h, batch._with(n), self._args_at, stream_handle(stream)) == _lib.F2K_OK

    def attend(self, Q, O, batch: PagedBatch, workspace, lse=None, stream=None) -> bool:
        """O = softmax(scale Q K^T) V of the batch's new tokens over the keys that they see; lse: fp32 [tokens, n_heads],
        the logarithm of the softmax's sum. O may be Q."""
        if self._rc:
            return False
        n = Q.shape[0]
        shape = n, self._heads, self._dim
        q, o = self._stride(Q, shape), self._stride(O, shape)
        if lse is not None:
            lse = self._vector(lse, torch.float32, (n, self._heads), "lse")
        if batch.index != self._index:
            raise TypeError("the batch lies on another device than the cache")
        size = 0
        if workspace is not None:
            size = workspace.nbytes
            if size and (workspace.get_device() != self._index or not workspace.is_contiguous()):
                raise TypeError("the workspace must be contiguous and on the cache's device")
        _ATTEND.pack_into(self._args, 0, Q.data_ptr(), O.data_ptr(), lse or 0, q, o, _p(workspace), size)
        return lib.f2k_kv_attend(self._h, batch._with(n), self._args_at, stream_handle(stream)) == _lib.F2K_OK
