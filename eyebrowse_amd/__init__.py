"""eyebrowse_amd: the eyebrowse attention hot path (prefill, decode, kv-write) on MI355X.

The compute lives in ``libeyebrowse_hip.so`` (hand-written gfx950 HIP kernels behind the C
ABI in ``include/eyebrowse_hip.h``); this package is a thin ctypes mirror of the
reference's Rust interface:

- ``gpu``: DType, EyebrowseError, Device, Tensor, Recorder (crates/eyebrowse-gpu);
- ``kernels``: attn_prefill, attn_decode, kv_write, rmsnorm, rope (crates/eyebrowse-kernels),
  linear_f16w (the projections around attention), plus chunked / windowed attention, the
  fused decode step and IEEE-half and OCP FP8 E4M3 caches; and a quantised model's operators:
  4-bit projections (linear_q4), block-scaled 8-bit caches (kv_write_i8, attn_*_i8), sampling;
  and the verification of a drafted tree (tree_plan, attn_tree, tree_accept, kv_compact, kv_fork);
- ``nn``: Linear, LinearQ4, Rope, KvCache, Attention (crates/eyebrowse-nn).
"""
from ._lib import LIB_PATH, lib
from .gpu import (DType, Device, DeviceUnavailable, EyebrowseError, Graph, LoadError,
                  OutOfMemory, Recorder, ShapeMismatch, Tensor, UnsupportedConfig)
from .kernels import (argmax, argmax_workspace_floats, attn_decode, attn_decode_step,
                      attn_decode_step_window, attn_decode_window, attn_decode_workspace_floats,
                      attn_prefill, attn_prefill_chunk, attn_prefill_fast,
                      attn_prefill_workspace_floats, launch_attn_prefill_fast,
                      attn_prefill_fast_workspace_floats, launch_attn_prefill_fast_ws,
                      kv_write, launch_argmax,
                      launch_attn_decode, launch_attn_decode_f16, launch_attn_decode_step,
                      launch_attn_decode_step_f16, launch_attn_decode_window,
                      launch_attn_prefill, launch_attn_prefill_chunk,
                      launch_attn_prefill_chunk_f16, launch_attn_prefill_chunk_ws,
                      launch_attn_prefill_ws, launch_kv_write, launch_kv_write_f16,
                      launch_attn_prologue, launch_attn_decode_step_noalloc,
                      launch_kv_write_f8, launch_attn_prefill_chunk_f8, launch_attn_decode_f8,
                      launch_attn_decode_step_f8,
                      attn_decode_noalloc_max_floats, launch_linear_f16w, launch_rmsnorm, launch_rope, linear_f16w,
                      linear_f16w_multi, linear_workspace_floats, rmsnorm, rope,
                      LANE_OPS_ROWS, launch_selftest_lane_ops, attn_prefill_pv16,
                      launch_attn_prefill_pv16, launch_attn_prefill_pv16_ws,
                      linear_q4, linear_q4_multi, linear_q4_workspace_floats, launch_linear_q4,
                      q4_packed_bytes, launch_q4_pack,
                      kv_write_i8, kv_read_i8, attn_decode_i8, attn_decode_step_i8,
                      attn_prefill_chunk_i8, attn_i8_workspace_floats, launch_kv_write_i8,
                      launch_kv_read_i8, launch_attn_decode_i8, launch_attn_prefill_chunk_i8,
                      sample, sample_workspace_floats, launch_sample,
                      TREE_MAX, tree_plan, attn_prologue_tree, attn_tree, attn_tree_i8,
                      attn_tree_workspace_floats, tree_accept, kv_compact, kv_fork,
                      launch_tree_plan, launch_tree_accept, launch_attn_prologue_tree,
                      launch_attn_tree, launch_attn_tree_i8)
from ._lib import CacheI8
from .nn import Attention, KvCache, Linear, LinearQ4, Rope

__all__ = [
    "LIB_PATH", "lib", "DType", "Device", "DeviceUnavailable", "EyebrowseError", "Graph",
    "LoadError", "argmax", "argmax_workspace_floats", "launch_argmax",
    "OutOfMemory", "Recorder", "ShapeMismatch", "Tensor", "UnsupportedConfig", "attn_decode",
    "attn_decode_step", "attn_decode_step_window", "attn_decode_window",
    "attn_decode_workspace_floats", "attn_prefill", "attn_prefill_chunk", "kv_write",
    "attn_prefill_fast", "launch_attn_prefill_fast", "attn_prefill_fast_workspace_floats",
    "launch_attn_prefill_fast_ws",
    "launch_attn_decode", "launch_attn_decode_f16", "launch_attn_decode_step",
    "launch_attn_decode_step_f16", "launch_attn_decode_window", "launch_attn_prefill",
    "launch_attn_prefill_chunk", "launch_attn_prefill_chunk_f16", "launch_attn_prefill_chunk_ws",
    "launch_attn_prefill_ws", "attn_prefill_workspace_floats", "launch_kv_write",
    "launch_kv_write_f16", "launch_kv_write_f8", "launch_attn_prefill_chunk_f8",
    "launch_attn_decode_f8", "launch_attn_decode_step_f8", "launch_linear_f16w", "linear_f16w", "linear_f16w_multi",
    "linear_workspace_floats", "launch_rmsnorm",
    "launch_rope", "launch_attn_prologue", "launch_attn_decode_step_noalloc",
    "attn_decode_noalloc_max_floats", "rmsnorm", "rope", "Attention", "KvCache", "Linear", "Rope",
    "LANE_OPS_ROWS", "launch_selftest_lane_ops", "attn_prefill_pv16", "launch_attn_prefill_pv16",
    "launch_attn_prefill_pv16_ws", "LinearQ4", "CacheI8",
    "linear_q4", "linear_q4_multi", "linear_q4_workspace_floats", "launch_linear_q4", "q4_packed_bytes", "launch_q4_pack",
    "kv_write_i8", "kv_read_i8", "attn_decode_i8", "attn_decode_step_i8",
    "attn_prefill_chunk_i8", "attn_i8_workspace_floats", "launch_kv_write_i8",
    "launch_kv_read_i8", "launch_attn_decode_i8", "launch_attn_prefill_chunk_i8", "sample",
    "sample_workspace_floats", "launch_sample",
    "TREE_MAX", "tree_plan", "attn_prologue_tree", "attn_tree", "attn_tree_i8",
    "attn_tree_workspace_floats", "tree_accept", "kv_compact", "kv_fork", "launch_tree_plan",
    "launch_tree_accept", "launch_attn_prologue_tree", "launch_attn_tree", "launch_attn_tree_i8",
]
