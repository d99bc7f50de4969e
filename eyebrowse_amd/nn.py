"""eyebrowse-nn pieces on the attention path over the C ABI: Rope, KvCache, RmsNorm
weights and the Attention forward between the projections.

Mirrors crates/eyebrowse-nn/src/{rope,kv_cache,attention}.rs. The q/k/v/o projections are
outside this path: ``Attention.forward_qkv`` starts from the projected q, k, v.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import numpy as np

from ._lib import AttentionDesc, Q4Weight, c_size, c_vp, lib
from .gpu import DType, Device, Recorder, Tensor, UnsupportedConfig, check
from .kernels import linear_f16w, linear_q4


class _Borrowed(Tensor):
    """A tensor owned by another object (rope tables, cache layers): never released here."""

    def __init__(self, handle: int, dev: Device, owner):
        super().__init__(handle, dev)
        self._owner = owner

    def release(self) -> None:
        self._h = c_vp()


class Rope:
    """Rope (crates/eyebrowse-nn/src/rope.rs:10-75): cos/sin tables [max_seq, hd/2]."""

    def __init__(self, handle: int, dev: Device, head_dim: int, max_seq: int):
        self._h = c_vp(handle)
        self.dev = dev
        self.head_dim = head_dim
        self.max_seq = max_seq

    @classmethod
    def build(cls, dev: Device, max_seq: int, head_dim: int, theta: float) -> "Rope":
        return cls.build_partial(dev, max_seq, head_dim, head_dim // 2, theta)

    @classmethod
    def build_partial(cls, dev: Device, max_seq: int, head_dim: int, rope_angles: int,
                      theta: float) -> "Rope":
        out = c_vp()
        check(lib().eb_rope_build_partial(dev.handle, max_seq, head_dim, rope_angles, theta,
                                          ctypes.byref(out)))
        return cls(out.value, dev, head_dim, max_seq)

    @property
    def handle(self):
        return self._h

    @property
    def cos(self) -> Tensor:
        return _Borrowed(lib().eb_rope_tables_cos(self._h), self.dev, self)

    @property
    def sin(self) -> Tensor:
        return _Borrowed(lib().eb_rope_tables_sin(self._h), self.dev, self)

    def apply(self, rec: Recorder, x: Tensor, seq: int, n_heads: int, base_pos: int) -> Tensor:
        out = c_vp()
        check(lib().eb_rope_apply(self._h, rec.handle, x.handle, seq, n_heads, base_pos,
                                  ctypes.byref(out)))
        return Tensor(out.value, self.dev)

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value:
            lib().eb_rope_tables_release(h)
            self._h = c_vp()


class Linear:
    """Linear (crates/eyebrowse-nn/src/linear.rs:5-23): bias-free, packed-f16 weight
    [out_f, in_f] (HF layout)."""

    def __init__(self, w: Tensor, in_f: int, out_f: int):
        self.w, self.in_f, self.out_f = w, in_f, out_f

    def forward(self, rec: Recorder, x: Tensor, rows: int) -> Tensor:
        out = Tensor.empty(rec.dev, (rows, self.out_f))
        linear_f16w(rec, x, self.w, out, rows, self.in_f, self.out_f)
        return out


class LinearQ4:
    """A bias-free projection with 4-bit codes and group scales (no counterpart in the reference):
    W[o, k] = (code[o, k] - zero[o, k // group]) * scale[o, k // group]. w: U32 [out_f, in_f / 8],
    eight codes per word along k, lowest bits first; scales: F16 [out_f, in_f / group]; zeros: U8 of
    that shape, or None (8 everywhere). group is 32, 64 or 128 and divides in_f. The weight is laid
    out once, into `packed`, as the kernels read it; w, scales and zeros are not kept, and are read
    when the constructor returns (it waits for earlier work on the null stream and the device's)."""

    def __init__(self, w: Tensor, scales: Tensor, zeros: Optional[Tensor], in_f: int, out_f: int,
                 group: int):
        out = c_vp()
        rec = Recorder(w.dev)
        check(lib().eb_q4_pack(rec.handle, w.handle, scales.handle,
                               zeros.handle if zeros is not None else None, in_f, out_f, group,
                               ctypes.byref(out)))
        self.packed = Tensor(out.value, w.dev)
        rec.submit()
        self.in_f, self.out_f, self.group, self.zeros = in_f, out_f, group, zeros is not None

    @property
    def desc(self) -> Q4Weight:
        return Q4Weight(self.packed.handle, self.in_f, self.out_f, self.group, int(self.zeros))

    @classmethod
    def from_f32(cls, dev: Device, weight, group: int = 128, symmetric: bool = True) -> "LinearQ4":
        """Round weight [out_f, in_f] to the nearest codes. Symmetric: scale = largest |w| of the
        group / 7, zero point 8; else scale = (largest - smallest) / 15 over the group and 0. A
        group whose scale no f16 holds (above 65504, or not finite) is refused."""
        w = np.asarray(weight, np.float32)
        out_f, in_f = w.shape
        if group not in (32, 64, 128) or in_f % group:
            raise UnsupportedConfig(f"LinearQ4: group {group} for in_f {in_f}")
        x = w.reshape(out_f, in_f // group, group)
        with np.errstate(over="ignore", invalid="ignore"):
            if symmetric:
                s = (np.abs(x).max(-1) / 7).astype(np.float16)
                z = np.full(s.shape, 8, np.uint8)
            else:
                lo, hi = np.minimum(x.min(-1), 0), np.maximum(x.max(-1), 0)
                s = ((hi - lo) / 15).astype(np.float16)
        if not np.isfinite(s).all():
            raise UnsupportedConfig("LinearQ4: a group's scale is not a finite f16")
        d = np.where(s > 0, s, 1).astype(np.float32)  # (a group of zeros: scale 0, any code)
        if not symmetric:
            z = np.clip(np.rint(-lo / d), 0, 15).astype(np.uint8)
        c = np.clip(np.rint(x / d[..., None]) + z[..., None], 0, 15).astype(np.uint32)
        c = c.reshape(out_f, in_f // 8, 8)
        words = np.bitwise_or.reduce(c << (4 * np.arange(8, dtype=np.uint32)), axis=-1)
        return cls(Tensor.from_array(dev, words.astype(np.uint32)), Tensor.from_array(dev, s),
                   None if symmetric else Tensor.from_array(dev, z), in_f, out_f, group)

    def forward(self, rec: Recorder, x: Tensor, rows: int) -> Tensor:
        out = Tensor.empty(rec.dev, (rows, self.out_f))
        linear_q4(rec, x, self, out, rows)
        return out


class KvCache:
    """KvCache (crates/eyebrowse-nn/src/kv_cache.rs:9-50): per-layer K/V tensors
    [max_seq, n_kv_heads, head_dims[l]]."""

    def __init__(self, handle: int, dev: Device, n_layers: int, max_seq: int, n_kv_heads: int,
                 dtype: DType = DType.F32):
        self._h = c_vp(handle)
        self.dev = dev
        self.max_seq = max_seq
        self.n_kv_heads = n_kv_heads
        self.dtype = dtype
        self.k = [_Borrowed(lib().eb_kv_cache_k(self._h, l), dev, self) for l in range(n_layers)]
        self.v = [_Borrowed(lib().eb_kv_cache_v(self._h, l), dev, self) for l in range(n_layers)]

    @classmethod
    def new(cls, dev: Device, n_layers: int, max_seq: int, n_kv_heads: int,
            head_dim: int, dtype: DType = DType.F32) -> "KvCache":
        return cls.new_per_layer(dev, [head_dim] * n_layers, max_seq, n_kv_heads, dtype)

    @classmethod
    def new_per_layer(cls, dev: Device, head_dims, max_seq: int, n_kv_heads: int,
                      dtype: DType = DType.F32) -> "KvCache":
        """dtype F32 is the reference's cache; F16 (IEEE half) halves and F8E4M3 (OCP FP8
        E4M3) quarters the cache bytes that decode streams (neither has a counterpart in
        the reference)."""
        arr = (c_size * max(1, len(head_dims)))(*head_dims)
        out = c_vp()
        check(lib().eb_kv_cache_new_per_layer_dtype(dev.handle, arr, len(head_dims), max_seq,
                                                    n_kv_heads, int(dtype), ctypes.byref(out)))
        return cls(out.value, dev, len(head_dims), max_seq, n_kv_heads, DType(dtype))

    @classmethod
    def new_i8(cls, dev: Device, n_layers: int, max_seq: int, n_kv_heads: int, head_dim: int,
               block: int = 64) -> "KvCache":
        """A block-scaled 8-bit cache (no counterpart in the reference): int8 codes and one
        power-of-two scale for each block of `block` rows and KV head; see new_i8_per_layer."""
        return cls.new_i8_per_layer(dev, [head_dim] * n_layers, max_seq, n_kv_heads, block)

    @classmethod
    def new_i8_per_layer(cls, dev: Device, head_dims, max_seq: int, n_kv_heads: int,
                         block: int = 64) -> "KvCache":
        """k[l], v[l]: I8 codes [max_seq, n_kv_heads, head_dims[l]]; k_scale[l], v_scale[l]: U8
        exponents e [ceil(max_seq / block), n_kv_heads]: a code stands for code * 2^(e - 127).
        block: a power of two from 16 to 256; head dims: multiples of 16 from 32 to 256."""
        arr = (c_size * max(1, len(head_dims)))(*head_dims)
        out = c_vp()
        check(lib().eb_kv_cache_new_i8(dev.handle, arr, len(head_dims), max_seq, n_kv_heads, block,
                                       ctypes.byref(out)))
        kv = cls(out.value, dev, len(head_dims), max_seq, n_kv_heads, DType.I8)
        kv.block = block
        kv.k_scale = [_Borrowed(lib().eb_kv_cache_k_scale(kv._h, l), dev, kv)
                      for l in range(len(head_dims))]
        kv.v_scale = [_Borrowed(lib().eb_kv_cache_v_scale(kv._h, l), dev, kv)
                      for l in range(len(head_dims))]
        return kv

    @property
    def handle(self):
        return self._h

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value:
            lib().eb_kv_cache_release(h)
            self._h = c_vp()


@dataclass
class Attention:
    """Attention (crates/eyebrowse-nn/src/attention.rs:10-23): head counts, scale, optional
    per-head q/k/v RMSNorm weights ([head_dim] f32 tensors) and, optionally, the four
    packed-f16 projections (all or none) with the model width `hidden`; or, with `hidden`, the four
    as 4-bit LinearQ4 in q4."""
    n_heads: int
    n_kv_heads: int
    head_dim: int
    scale: float
    q_norm: Optional[Tensor] = None
    k_norm: Optional[Tensor] = None
    v_norm: Optional[Tensor] = None
    norm_eps: float = 1e-6
    window: int = 0  # sliding window of a local layer (0: global attention)
    q_proj: Optional[Tensor] = None  # [n_heads*head_dim, hidden]
    k_proj: Optional[Tensor] = None  # [n_kv_heads*head_dim, hidden]
    v_proj: Optional[Tensor] = None
    o_proj: Optional[Tensor] = None  # [hidden, n_heads*head_dim]
    hidden: int = 0
    q4: Optional[tuple] = None  # (q, k, v, o) LinearQ4; q, k and v share group and zero points

    def __post_init__(self):
        h = lambda t: t.handle if t is not None else None  # noqa: E731
        d = AttentionDesc(self.n_heads, self.n_kv_heads, self.head_dim, self.scale, self.norm_eps,
                          h(self.q_norm), h(self.k_norm), h(self.v_norm), self.window,
                          h(self.q_proj), h(self.k_proj), h(self.v_proj), h(self.o_proj),
                          self.hidden)
        out = c_vp()
        if self.q4 is not None:
            q, k, v, o = self.q4
            proj = (Q4Weight * 4)(q.desc, k.desc, v.desc, o.desc)
            check(lib().eb_attention_new_q4(ctypes.byref(d), proj, ctypes.byref(out)))
        else:
            check(lib().eb_attention_new(ctypes.byref(d), ctypes.byref(out)))
        self._h = out

    def forward_qkv(self, rec: Recorder, q: Tensor, k: Tensor, v: Tensor, rope: Rope,
                    kv: KvCache, layer: int, rows: int, base_pos: int) -> Tensor:
        """Attention::forward (attention.rs:30-185) from the projected q [rows, H*hd],
        k/v [rows, Hkv*hd]: norms, RoPE, kv_write, then prefill (base_pos == 0 and
        rows > 1), chunked prefill over the cache (base_pos > 0 and rows > 1) or the fused
        decode step (rows == 1). Returns [rows, H*hd], the o_proj input."""
        out = c_vp()
        check(lib().eb_attention_forward_qkv(self._h, rec.handle, q.handle, k.handle, v.handle,
                                             rope.handle, kv.handle, layer, rows, base_pos,
                                             ctypes.byref(out)))
        return Tensor(out.value, rec.dev)

    def forward(self, rec: Recorder, x: Tensor, rope: Rope, kv: KvCache, layer: int, rows: int,
                base_pos: int) -> Tensor:
        """Attention::forward (attention.rs:30-45) whole: x [rows, hidden] -> [rows, hidden]
        (q/k/v projections in one launch, forward_qkv, o_proj)."""
        out = c_vp()
        check(lib().eb_attention_forward(self._h, rec.handle, x.handle, rope.handle, kv.handle,
                                         layer, rows, base_pos, ctypes.byref(out)))
        return Tensor(out.value, rec.dev)

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value:
            lib().eb_attention_release(h)
            self._h = c_vp()
