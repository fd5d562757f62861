"""torch custom ops over the C ABI: `torch.ops.hkv.write`, `torch.ops.hkv.decode`, `torch.ops.hkv.combine`, those of a
bounded cache: `decode_window`, `prefill_window`, `accumulate_weights`, `evict`, the write that rotates (`write_rotary`) and those of the
8-bit cache: `write_b8`, `write_rotary_b8`, `decode_b8`, `prefill_b8`.

`write_rotary` and `write_rotary_b8` take the query as their query_out too, as torch's own ops take an input as out=: their schemas
name query_out as what is written. A front end that gives mutated arguments as copies turns the copy, from the query as it was.

The ops are thin: they pass the tensors' device pointers, the strides and the current CUDA stream to `libhkv.so`
(include/hkv.h) and mutate their output arguments in place, like the reference's TileLang-launched kernels mutate the
cache and the output buffer (kv_fp4_serving.py:994-1005, :894-915 in the reference). Registering them with torch lets
graph-capturing front ends (torch.compile, vLLM's piecewise graphs) treat the launches as opaque mutating ops. There is
a CUDA implementation only: calling an op with CPU tensors raises. `combine` is kept for the reference's three-launch
sequence; the merge of split sequences runs inside `decode`, so it launches nothing.
"""
import ctypes as C

import torch

from . import _lib
from . import kernels as K

_REGISTERED = False


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _p(t):
    return C.c_void_p(t.data_ptr())


def _strides6(strides):
    if len(strides) != 6:
        raise ValueError("strides must be (data page, data position, data head, scale page, scale position, scale head)")
    return tuple(int(x) for x in strides)


def _rows(rows):
    if len(rows) % 4:
        raise ValueError("rows: four numbers per request (table row, first query token, one past the last, context)")
    return [tuple(int(x) for x in rows[i:i + 4]) for i in range(0, len(rows), 4)]


def _strides2(strides):
    if len(strides) != 2:
        raise ValueError("strides of the 8-bit cache must be (page, head)")
    return tuple(int(x) for x in strides)


def register():
    """defines the hkv::* ops once per process; returns torch.ops.hkv"""
    global _REGISTERED
    if _REGISTERED:
        return torch.ops.hkv
    lib = torch.library.Library("hkv", "DEF")
    lib.define("write(Tensor key, Tensor value, Tensor(a!) k_data, Tensor(b!) k_sf, Tensor(c!) v_data, Tensor(d!) v_sf, "
               "int[] strides, int page_size, Tensor slot_mapping, Tensor gk, Tensor gv, bool search) -> ()")
    lib.define("decode(Tensor query, Tensor k_data, Tensor k_sf, Tensor v_data, Tensor v_sf, int[] strides, int page_size, "
               "Tensor block_tables, Tensor seq_lens, Tensor query_start_loc, float sm_scale, float v_scale, Tensor gk, "
               "Tensor gv, int qlmax, Tensor(a!) workspace, int splits, Tensor(b!) out) -> ()")
    lib.define("combine(Tensor(a!) workspace, Tensor query_start_loc, int num_kv_heads, int group, int head_dim, int qlmax, "
               "float v_scale, Tensor(b!) out) -> ()")

    cache = "Tensor k_data, Tensor k_sf, Tensor v_data, Tensor v_sf, int[] strides, int page_size, Tensor block_tables, "
    lib.define("decode_window(Tensor query, " + cache + "Tensor seq_lens, Tensor query_start_loc, float sm_scale, float v_scale, "
               "Tensor gk, Tensor gv, int qlmax, Tensor(a!) workspace, int splits, int window, int sinks, Tensor? signs, bool k8, "
               "Tensor(b!) out, Tensor(c!)? lse) -> ()")
    lib.define("prefill_window(Tensor query, " + cache + "int[] rows, float qk_scale, float out_scale, int num_kv_heads, int chunk, "
               "int window, int sinks, Tensor? signs, bool k8, Tensor(a!) out, Tensor(b!)? lse) -> ()")
    lib.define("accumulate_weights(Tensor query, " + cache + "Tensor seq_lens, Tensor query_start_loc, float sm_scale, Tensor gk, "
               "int qlmax, Tensor lse, int window, int sinks, Tensor? signs, bool k8, Tensor(a!) weights) -> ()")
    lib.define("evict(Tensor(a!) k_data, Tensor(b!) k_sf, Tensor(c!) v_data, Tensor(d!) v_sf, int[] strides, int page_size, "
               "int head_dim, Tensor block_tables, Tensor seq_lens, Tensor(e!) weights, int keep, int sinks, int recent, "
               "Tensor(f!) kept, Tensor(g!) out_lens, Tensor? out_tables, Tensor(h!)? out_weights, bool k8) -> ()")

    turn = "Tensor positions, Tensor cos_sin, Tensor gk, Tensor gv, bool interleaved, "
    tiles = "Tensor(a!) k_tiles, Tensor(b!) v_tiles, int[] strides, int page_size, Tensor slot_mapping, "
    lib.define("write_rotary(Tensor query, Tensor key, Tensor value, Tensor(a!) k_data, Tensor(b!) k_sf, Tensor(c!) v_data, Tensor(d!) v_sf, "
               "int[] strides, int page_size, Tensor slot_mapping, " + turn + "bool search, Tensor? signs, bool k8, Tensor(e!) query_out) -> ()")
    lib.define("write_b8(Tensor key, Tensor value, " + tiles + "Tensor gk, Tensor gv, str fmt) -> ()")
    lib.define("write_rotary_b8(Tensor query, Tensor key, Tensor value, " + tiles + turn + "str fmt, Tensor(c!) query_out) -> ()")
    tiles = "Tensor k_tiles, Tensor v_tiles, int[] strides, int page_size, Tensor block_tables, "
    lib.define("decode_b8(Tensor query, " + tiles + "Tensor seq_lens, Tensor query_start_loc, float sm_scale, float v_scale, Tensor gk, "
               "Tensor gv, int qlmax, Tensor(a!) workspace, int splits, str fmt, int window, int sinks, Tensor(b!) out, "
               "Tensor(c!)? lse) -> ()")
    lib.define("prefill_b8(Tensor query, " + tiles + "int[] rows, float qk_scale, float out_scale, int num_kv_heads, int chunk, str fmt, "
               "int window, int sinks, Tensor(a!) out, Tensor(b!)? lse) -> ()")

    # the implementations go through the host wrappers of kernels.py, so dtypes, contiguity and shapes are checked
    # once, in one place, before any pointer reaches the C ABI
    def write(key, value, k_data, k_sf, v_data, v_sf, strides, page_size, slot_mapping, gk, gv, search):
        K.write(key, value, (k_data, k_sf, v_data, v_sf), _strides6(strides), int(page_size), slot_mapping, gk, gv,
                bool(search))

    def decode(query, k_data, k_sf, v_data, v_sf, strides, page_size, block_tables, seq_lens, query_start_loc, sm_scale,
               v_scale, gk, gv, qlmax, workspace, splits, out):
        if block_tables.dim() != 2 or query_start_loc.shape[0] != block_tables.shape[0] + 1 or \
                seq_lens.shape[0] != block_tables.shape[0]:
            raise ValueError("block_tables (B, MP), seq_lens (B,), query_start_loc (B + 1,)")
        K.decode_ragged(query, (k_data, k_sf, v_data, v_sf), _strides6(strides), int(page_size), block_tables, seq_lens,
                        query_start_loc, float(sm_scale), float(v_scale), gk, gv, int(qlmax), out, workspace,
                        splits=int(splits) or None)

    def combine(workspace, query_start_loc, num_kv_heads, group, head_dim, qlmax, v_scale, out):
        K._need_cuda(workspace, query_start_loc, out)
        with torch.cuda.device(out.device):
            rc = _lib.load().hkv_combine(_p(workspace), workspace.numel() * workspace.element_size(), _p(query_start_loc),
                                         query_start_loc.shape[0] - 1, int(num_kv_heads), int(group), int(head_dim),
                                         int(qlmax), float(v_scale), _p(out), _stream())
        _lib.check(rc, "hkv_combine")

    def decode_window(query, k_data, k_sf, v_data, v_sf, strides, page_size, block_tables, seq_lens, query_start_loc, sm_scale,
                      v_scale, gk, gv, qlmax, workspace, splits, window, sinks, signs, k8, out, lse):
        K.decode_window(query, (k_data, k_sf, v_data, v_sf), _strides6(strides), int(page_size), block_tables, seq_lens,
                        query_start_loc, float(sm_scale), float(v_scale), gk, gv, int(qlmax), out, workspace, int(window), int(sinks),
                        splits=int(splits) or None, signs=signs, k8=bool(k8), lse=lse)

    def prefill_window(query, k_data, k_sf, v_data, v_sf, strides, page_size, block_tables, rows, qk_scale, out_scale, num_kv_heads,
                       chunk, window, sinks, signs, k8, out, lse):
        K.prefill_window(query, (k_data, k_sf, v_data, v_sf), _strides6(strides), int(page_size), block_tables, _rows(rows), float(qk_scale),
                         float(out_scale), int(num_kv_heads), out, int(window), int(sinks), chunk=int(chunk), signs=signs, k8=bool(k8),
                         lse=lse)

    def accumulate_weights(query, k_data, k_sf, v_data, v_sf, strides, page_size, block_tables, seq_lens, query_start_loc, sm_scale,
                           gk, qlmax, lse, window, sinks, signs, k8, weights):
        K.accumulate_weights(query, (k_data, k_sf, v_data, v_sf), _strides6(strides), int(page_size), block_tables, seq_lens,
                             query_start_loc, float(sm_scale), gk, int(qlmax), lse, weights, window=int(window), sinks=int(sinks),
                             signs=signs, k8=bool(k8))

    def evict(k_data, k_sf, v_data, v_sf, strides, page_size, head_dim, block_tables, seq_lens, weights, keep, sinks, recent, kept,
              out_lens, out_tables, out_weights, k8):
        K.evict((k_data, k_sf, v_data, v_sf), _strides6(strides), int(page_size), int(head_dim), block_tables, seq_lens, weights,
                int(keep), int(sinks), int(recent), kept, out_lens, out_tables=out_tables, out_weights=out_weights, k8=bool(k8))

    def write_rotary(query, key, value, k_data, k_sf, v_data, v_sf, strides, page_size, slot_mapping, positions, cos_sin, gk, gv,
                     interleaved, search, signs, k8, query_out):
        K.write_rotary(query, key, value, (k_data, k_sf, v_data, v_sf), _strides6(strides), int(page_size), slot_mapping, positions, cos_sin,
                       gk, gv, query_out, interleaved=bool(interleaved), search=bool(search), signs=signs, k8=bool(k8))

    def write_b8(key, value, k_tiles, v_tiles, strides, page_size, slot_mapping, gk, gv, fmt):
        K.write_b8(key, value, (k_tiles, v_tiles), _strides2(strides), int(page_size), slot_mapping, gk, gv, fmt=fmt)

    def write_rotary_b8(query, key, value, k_tiles, v_tiles, strides, page_size, slot_mapping, positions, cos_sin, gk, gv, interleaved,
                        fmt, query_out):
        K.write_rotary_b8(query, key, value, (k_tiles, v_tiles), _strides2(strides), int(page_size), slot_mapping, positions, cos_sin, gk, gv,
                          query_out, interleaved=bool(interleaved), fmt=fmt)

    def decode_b8(query, k_tiles, v_tiles, strides, page_size, block_tables, seq_lens, query_start_loc, sm_scale, v_scale, gk, gv, qlmax,
                  workspace, splits, fmt, window, sinks, out, lse):
        K.decode_b8(query, (k_tiles, v_tiles), _strides2(strides), int(page_size), block_tables, seq_lens, query_start_loc,
                    float(sm_scale), float(v_scale), gk, gv, int(qlmax), out, workspace, fmt=fmt, window=int(window), sinks=int(sinks),
                    splits=int(splits) or None, lse=lse)

    def prefill_b8(query, k_tiles, v_tiles, strides, page_size, block_tables, rows, qk_scale, out_scale, num_kv_heads, chunk, fmt,
                   window, sinks, out, lse):
        K.prefill_b8(query, (k_tiles, v_tiles), _strides2(strides), int(page_size), block_tables, _rows(rows), float(qk_scale),
                     float(out_scale), int(num_kv_heads), out, fmt=fmt, window=int(window), sinks=int(sinks), chunk=int(chunk), lse=lse)

    for f in (write_rotary, write_b8, write_rotary_b8, decode_b8, prefill_b8):
        lib.impl(f.__name__, f, "CUDA")
    lib.impl("write", write, "CUDA")
    lib.impl("decode_window", decode_window, "CUDA")
    lib.impl("prefill_window", prefill_window, "CUDA")
    lib.impl("accumulate_weights", accumulate_weights, "CUDA")
    lib.impl("evict", evict, "CUDA")
    lib.impl("decode", decode, "CUDA")
    lib.impl("combine", combine, "CUDA")
    register._lib = lib                       # keep the Library object alive
    _REGISTERED = True
    return torch.ops.hkv
