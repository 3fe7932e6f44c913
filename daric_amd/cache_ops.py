"""`daric.cache_ops` API on the gfx950 HIP library.

Drop-in for the reference's pybind11 module (stub daric/cache_ops.pyi:1-53,
bindings csrc/cache_ops/bindings.cpp:7-31): `CacheCopier` with
register_layer / register_store / gather_pages / scatter_pages, and the free
functions batched_memcpy_d2h / batched_memcpy_h2d keep their signatures,
argument meaning and errors (RuntimeError with the reference's message text).

Additions (no reference counterpart; the .pyi grows, nothing changes):
  CacheCopier.register_k_scale, CacheCopier.scatter_pages_rerotate (and its
  allocation-free form scatter_pages_rerotate_noalloc),
  CacheCopier.gather_tokens / scatter_tokens (token-major staging for any
  cache layout), rerotate_pages, kv_deviation, topk_per_chunk, merge_rows,
  select_merge (the three selection calls in one), attend_pages (attention
  over the paged cache), weigh_tokens and evict_tokens (eviction by
  accumulated attention weight), rotate_rows and append_tokens (new rows, rotated
  into the cache), select_beams and reorder_beams (beam search over it), kernel
  timing.

Every call is asynchronous on `stream` (0 = the current torch stream of the
first layer's device, as in reference copier.cpp:27-30). The wrapper keeps
strong references to registered tensors (copier.cpp:10, 21-24) and records
temporary inputs on the launch stream (kernels.cu:202, copier.cpp:69).
"""
from __future__ import annotations

import array
import ctypes
import struct
from collections.abc import Sequence
from contextlib import nullcontext
from itertools import chain
from operator import attrgetter
from typing import Optional

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import I64, DaricChunk, DaricRope, check, desc, layer_views, load, str_array, views

__all__ = [
    "CacheCopier", "batched_memcpy_d2h", "batched_memcpy_h2d", "rerotate_pages",
    "kv_deviation", "topk_per_chunk", "merge_rows", "select_merge", "SELECT_KEYS_READY",
    "SELECT_ONE_PASS", "attend_pages", "weigh_tokens", "evict_tokens", "rotate_rows", "append_tokens",
    "select_beams", "reorder_beams", "timing_enable", "timing_read",
]


# The current stream's raw handle without building a torch.cuda.Stream object
# (0.1 us against 2 us per call on MI355X); the public call is the fallback.
_RAW_STREAM = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _resolve_stream(stream: int, device: Optional[torch.device]) -> int:
    if stream:
        return int(stream)
    if device is None or device.type != "cuda":
        return 0
    if _RAW_STREAM is not None:
        idx = device.index if device.index is not None else torch.cuda.current_device()
        return int(_RAW_STREAM(idx))
    return torch.cuda.current_stream(device).cuda_stream


_EXT_STREAMS: dict = {}


def _ext_stream(stream: int, device: torch.device):
    key = (int(stream), device.index)
    s = _EXT_STREAMS.get(key)
    if s is None:
        if len(_EXT_STREAMS) > 64:
            _EXT_STREAMS.clear()
        s = _EXT_STREAMS[key] = torch.cuda.ExternalStream(stream, device=device)
    return s


def _on_stream(stream: int, device: torch.device):
    """Context in which torch allocates and launches on `stream`; none to enter
    where that is the current stream already (entering two of them was most of
    what made a selection over 96 chunks 80 us on the host, now 63 us)."""
    if stream == _resolve_stream(0, device):
        return nullcontext()
    return torch.cuda.stream(_ext_stream(stream, device))


_HERE = nullcontext()


# Whether tensors may have forward-mode tangents. Where torch does not tell, they may:
# asking each tensor takes a microsecond.
if hasattr(forward_ad, "_current_level"):
    def _in_dual_level() -> bool:
        return forward_ad._current_level >= 0
else:
    def _in_dual_level() -> bool:
        return True


_REQUIRES_GRAD = attrgetter("requires_grad")


def _record(stream: int, device: torch.device, *tensors) -> None:
    """Keep caching-allocator memory of temporaries alive until `stream` has
    consumed them (the reference's record_tensor_on_external_stream). Not
    while a graph is being captured: a captured graph's inputs must outlive
    its replays, which is the caller's to ensure, as for any graph."""
    if device is None or device.type != "cuda" or torch.cuda.is_current_stream_capturing():
        return
    ext = _ext_stream(stream, device)
    for t in tensors:
        if t is not None and t.is_cuda:
            t.record_stream(ext)


def _rope(inv_freq: torch.Tensor, rotary_dim: int, is_neox_style: bool, device) -> DaricRope:
    if not isinstance(inv_freq, torch.Tensor) or not inv_freq.is_cuda:
        raise RuntimeError("inv_freq must be a float32 device tensor")
    if inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous():
        raise RuntimeError("inv_freq must be a contiguous float32 tensor")
    if inv_freq.numel() < int(rotary_dim) // 2:
        raise RuntimeError(f"inv_freq has {inv_freq.numel()} entries, rotary_dim/2 = {int(rotary_dim) // 2}")
    if device is not None and inv_freq.device != device:
        raise RuntimeError("inv_freq must be on the KV cache's device")
    r = DaricRope()
    r.inv_freq = inv_freq.data_ptr()
    r.rotary_dim = int(rotary_dim)
    r.is_neox = 1 if is_neox_style else 0
    return r


class CacheCopier:
    """Staged KV-cache gather/scatter (reference csrc/cache_ops/copier.cpp)."""

    def __init__(self) -> None:
        self._lib = load()
        h = ctypes.c_void_p()
        check(self._lib.daric_copier_create(ctypes.byref(h)))
        self._h = h
        self._layers: dict[str, torch.Tensor] = {}
        self._scales: dict[str, torch.Tensor] = {}
        self._store: Optional[torch.Tensor] = None

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value:
            self._lib.daric_copier_destroy(h)
            self._h = None

    # -------------------------------------------------------------- register
    def register_layer(self, name: str, tensor: torch.Tensor, is_page_first: bool) -> None:
        d = desc(tensor)
        check(self._lib.daric_copier_register_layer(self._h, str(name).encode(), ctypes.byref(d),
                                                    1 if is_page_first else 0))
        self._layers[str(name)] = tensor

    def register_store(self, buffer: torch.Tensor) -> None:
        d = desc(buffer)
        check(self._lib.daric_copier_register_store(self._h, ctypes.byref(d)))
        self._store = buffer

    def register_k_scale(self, name: str, k_scale: Optional[torch.Tensor]) -> None:
        """Per-head fp32 K scales of an fp8 layer (None clears them)."""
        d = desc(k_scale) if k_scale is not None else None
        check(self._lib.daric_copier_register_k_scale(
            self._h, str(name).encode(), ctypes.byref(d) if d is not None else None))
        if k_scale is None:
            self._scales.pop(str(name), None)
        else:
            self._scales[str(name)] = k_scale

    # -------------------------------------------------------------- copies
    def _device(self, layer_names) -> Optional[torch.device]:
        if len(layer_names) == 0:
            return None
        t = self._layers.get(str(layer_names[0]))
        return t.device if t is not None else None

    def _copy(self, fn, layer_names, offsets, byte_sizes, indices_flat, indices_offsets, stream,
              extra=(), record=()):
        names = list(layer_names)
        dev = self._device(names)
        st = _resolve_stream(stream, dev)
        idx = desc(indices_flat)
        off, sz, ioff = I64(offsets), I64(byte_sizes), I64(indices_offsets)
        status = fn(self._h, str_array(names), len(names), off.ptr, off.n, sz.ptr, sz.n,
                    ctypes.byref(idx), ioff.ptr, ioff.n, *extra, ctypes.c_uint64(st))
        check(status)
        if names:
            _record(st, dev, indices_flat, *record)

    def gather_pages(self, layer_names: Sequence[str], offsets: Sequence[int],
                     byte_sizes: Sequence[int], indices_flat: torch.Tensor,
                     indices_offsets: Sequence[int], stream: int = 0) -> None:
        self._copy(self._lib.daric_copier_gather_pages, layer_names, offsets, byte_sizes,
                   indices_flat, indices_offsets, stream)

    def scatter_pages(self, layer_names: Sequence[str], offsets: Sequence[int],
                      byte_sizes: Sequence[int], indices_flat: torch.Tensor,
                      indices_offsets: Sequence[int], stream: int = 0) -> None:
        self._copy(self._lib.daric_copier_scatter_pages, layer_names, offsets, byte_sizes,
                   indices_flat, indices_offsets, stream)

    def gather_tokens(self, layer_names: Sequence[str], offsets: Sequence[int],
                      byte_sizes: Sequence[int], indices_flat: torch.Tensor,
                      indices_offsets: Sequence[int], stream: int = 0) -> None:
        """gather_pages into token-major rows: job i's store range becomes
        [n_kv][n_sel * PS][H][D] (K rows then V rows) for any cache layout
        (see include/daric_cache_ops.h). byte_sizes[i] = n_kv * n_sel * PS *
        H * D * element size. No counterpart in the reference."""
        self._copy(self._lib.daric_copier_gather_tokens, layer_names, offsets, byte_sizes,
                   indices_flat, indices_offsets, stream)

    def scatter_tokens(self, layer_names: Sequence[str], offsets: Sequence[int],
                       byte_sizes: Sequence[int], indices_flat: torch.Tensor,
                       indices_offsets: Sequence[int], stream: int = 0) -> None:
        """Inverse of gather_tokens. No counterpart in the reference."""
        self._copy(self._lib.daric_copier_scatter_tokens, layer_names, offsets, byte_sizes,
                   indices_flat, indices_offsets, stream)

    def scatter_pages_rerotate(self, layer_names: Sequence[str], offsets: Sequence[int],
                               byte_sizes: Sequence[int], indices_flat: torch.Tensor,
                               indices_offsets: Sequence[int], deltas: Sequence[int],
                               num_tokens: Sequence[int], inv_freq: torch.Tensor,
                               rotary_dim: int, is_neox_style: bool = True,
                               stream: int = 0) -> None:
        """scatter_pages + re-rotation of the first num_tokens[i] tokens of job
        i by deltas[i] positions, in one pass (see include/daric_cache_ops.h)."""
        self._fused(self._lib.daric_copier_scatter_pages_rerotate, layer_names, offsets, byte_sizes,
                    indices_flat, indices_offsets, deltas, num_tokens, inv_freq, rotary_dim,
                    is_neox_style, stream)

    def scatter_pages_rerotate_noalloc(self, layer_names: Sequence[str], offsets: Sequence[int],
                                       byte_sizes: Sequence[int], indices_flat: torch.Tensor,
                                       indices_offsets: Sequence[int], deltas: Sequence[int],
                                       num_tokens: Sequence[int], inv_freq: torch.Tensor,
                                       rotary_dim: int, is_neox_style: bool = True,
                                       stream: int = 0) -> None:
        """scatter_pages_rerotate without allocating device or pinned memory:
        large job lists are staged in a static per-GPU array of 3276 jobs.
        Calls that overlap on one GPU race on that array (see
        include/daric_cache_ops.h). No counterpart in the reference."""
        self._fused(self._lib.daric_copier_scatter_pages_rerotate_noalloc, layer_names, offsets,
                    byte_sizes, indices_flat, indices_offsets, deltas, num_tokens, inv_freq,
                    rotary_dim, is_neox_style, stream)

    def _fused(self, fn, layer_names, offsets, byte_sizes, indices_flat, indices_offsets, deltas,
               num_tokens, inv_freq, rotary_dim, is_neox_style, stream):
        names = list(layer_names)
        if len(deltas) != len(names) or len(num_tokens) != len(names):
            if names:
                raise RuntimeError("deltas and num_tokens must have one entry per job")
        dev = self._device(names)
        rope = _rope(inv_freq, rotary_dim, is_neox_style, dev) if names else DaricRope()
        dl, nt = I64(deltas), I64(num_tokens)
        self._copy(fn, names, offsets, byte_sizes, indices_flat, indices_offsets, stream,
                   extra=(dl.ptr, nt.ptr, ctypes.byref(rope)), record=(inv_freq,))


def _memcpy(fn, dev_t, host_t, dev_offsets, host_offsets, sizes, stream, d2h):
    n = len(sizes)
    if len(dev_offsets) != n or len(host_offsets) != n:
        raise RuntimeError("offset and size lists must have the same length")
    if n == 0:
        return
    dev = dev_t.device if dev_t.is_cuda else None
    st = _resolve_stream(stream, dev)
    a, b = desc(dev_t), desc(host_t)
    do, ho, sz = I64(dev_offsets), I64(host_offsets), I64(sizes)
    if d2h:
        check(fn(ctypes.byref(a), ctypes.byref(b), do.ptr, ho.ptr, sz.ptr, n, ctypes.c_uint64(st)))
    else:
        check(fn(ctypes.byref(b), ctypes.byref(a), ho.ptr, do.ptr, sz.ptr, n, ctypes.c_uint64(st)))


def batched_memcpy_d2h(staging: torch.Tensor, shm: torch.Tensor, stg_offsets: Sequence[int],
                       shm_offsets: Sequence[int], sizes: Sequence[int], stream: int = 0) -> None:
    """One hipMemcpyAsync per (stg_offset, shm_offset, size) region (reference
    helpers.cu:187-217). shm must be page-locked host memory."""
    _memcpy(load().daric_batched_memcpy_d2h, staging, shm, stg_offsets, shm_offsets, sizes, stream, True)


def batched_memcpy_h2d(shm: torch.Tensor, staging: torch.Tensor, shm_offsets: Sequence[int],
                       stg_offsets: Sequence[int], sizes: Sequence[int], stream: int = 0) -> None:
    """Mirror of batched_memcpy_d2h (reference helpers.cu:219-248)."""
    _memcpy(load().daric_batched_memcpy_h2d, staging, shm, stg_offsets, shm_offsets, sizes, stream, False)


_LAYER_ARRAYS: dict = {}


def _layer_array(layers: Sequence[torch.Tensor]):
    """daric_tensor array of `layers`, cached per (address, shape, strides,
    dtype, device) signature: callers pass the same cache tensors every call."""
    key = tuple((t.data_ptr(), t.shape, t.stride(), t.dtype, t.device) for t in layers)
    arr = _LAYER_ARRAYS.get(key)
    if arr is None:
        arr = (_lib.DaricTensor * max(len(layers), 1))()
        for i, t in enumerate(layers):
            arr[i] = desc(t)
        if len(_LAYER_ARRAYS) >= 64:
            _LAYER_ARRAYS.clear()
        _LAYER_ARRAYS[key] = arr
    return arr


def _segments(segs):
    """(address of daric_rope_segment[n], n, keep-alive) of a list of 4-tuples
    of ints, or of what else numpy takes as rows of four int64 values. Without a
    Python-level loop: 4, 100 and 1000 tuples take 0.8, 7.0 and 63 us on the
    host, through numpy 1.5, 10.8 and 95 (with a generator over the tuples 0.9,
    11.8 and 111)."""
    if set(map(type, segs)) == {tuple} and set(map(len, segs)) == {4}:
        try:
            flat = array.array("q", list(chain.from_iterable(segs)))
            return flat.buffer_info()[0], len(segs), flat
        except TypeError:       # not ints: numpy converts or refuses them
            pass
    a = np.ascontiguousarray(np.asarray(segs, dtype=np.int64).reshape(-1, 4))
    return a.ctypes.data, len(segs), a


def rerotate_pages(layers: Sequence[torch.Tensor], page_first: bool, block_table: torch.Tensor,
                   segments: Sequence[tuple[int, int, int, int]], inv_freq: torch.Tensor,
                   rotary_dim: int, is_neox_style: bool = True,
                   k_scales: Optional[torch.Tensor] = None, stream: int = 0) -> None:
    """In-place re-rotation of the K rows of every segment
    (bt_offset, tok_start, n_tokens, delta) in every layer: the counterpart of
    the reference's per-layer _launch_triton_rerotate (adapter.py:297-396).
    k_scales ([L, H] fp32, positive) is checked but leaves the result
    unchanged: fp8 codes are rotated as stored, since a per-head scale cancels
    in a linear rotation (the reference's kernel rotates the raw fp8 values)."""
    layers = list(layers)
    segs = list(segments)
    if not layers or not segs:
        return
    dev = layers[0].device
    st = _resolve_stream(stream, dev)
    rope = _rope(inv_freq, rotary_dim, is_neox_style, dev)
    sarr, n_segs, _keep = _segments(segs)
    bt = desc(block_table)
    ks = desc(k_scales) if k_scales is not None else None
    check(load().daric_rerotate_pages(_layer_array(layers), len(layers), 1 if page_first else 0,
                                      ctypes.byref(bt), sarr, n_segs, ctypes.byref(rope),
                                      ctypes.byref(ks) if ks is not None else None,
                                      ctypes.c_uint64(st)))
    _record(st, dev, block_table, inv_freq, k_scales)


def _chunks(chunks):
    """(pointer to daric_chunk[n], n, keep-alive) from a sequence of
    (bt_offset, row_offset, n_tokens, k[, tok_start]) tuples or an int64
    [n, 4] / [n, 5] array; tok_start defaults to 0."""
    a = np.asarray(chunks, dtype=np.int64)
    if a.size == 0:
        a = np.zeros((1, 5), np.int64)
        return ctypes.cast(a.ctypes.data, ctypes.POINTER(DaricChunk)), 0, a
    if a.ndim != 2 or a.shape[1] not in (4, 5):
        raise ValueError("chunks must be (bt_offset, row_offset, n_tokens, k[, tok_start]) entries")
    if a.shape[1] == 4:
        a = np.concatenate([a, np.zeros((a.shape[0], 1), np.int64)], axis=1)
    a = np.ascontiguousarray(a)
    return ctypes.cast(a.ctypes.data, ctypes.POINTER(DaricChunk)), a.shape[0], a


def _new_keys(st: int, dev, n_layers: int, rows: int, chunks: np.ndarray) -> torch.Tensor:
    """Deviation keys [n_layers, rows] allocated on stream `st`. Rows outside
    every chunk are 0, by a fill ordered before the kernel; chunks that follow
    each other over all rows, as a batch's plan does, leave none, and the kernel
    writes every row of a chunk (0 for a block id out of range): no fill then
    (a call over 294 rows of 17 layers 43.2 -> 41.4 us, over 49152 rows of 32
    layers 1335 -> 1332 us on MI355X)."""
    begin = chunks[:, 1]
    end = begin + chunks[:, 2]
    whole = begin[0] == 0 and end[-1] == rows and bool((begin[1:] == end[:-1]).all())
    with _on_stream(st, dev):
        return (torch.empty if whole else torch.zeros)((n_layers, rows), dtype=torch.float32, device=dev)


def kv_deviation(layers: Sequence[torch.Tensor], page_first: bool, block_table: torch.Tensor,
                 k_new: torch.Tensor, chunks, keys: Optional[torch.Tensor] = None,
                 stream: int = 0, k_scales: Optional[torch.Tensor] = None) -> torch.Tensor:
    """keys[l, row] = sum over (h, d) of (k_new - cached K)^2 in the fixed
    order of daric_amd/csrc/select_kernels.hip. chunks: (bt_offset,
    row_offset, n_tokens, k[, tok_start]); token j of a chunk is token
    tok_start + j of the block list at block_table[bt_offset]. k_scales: [L, H] fp32 per-head scales of an fp8
    cache (None: scale 1)."""
    layers = list(layers)
    dev = layers[0].device
    st = _resolve_stream(stream, dev)
    carr, n, ch = _chunks(chunks)
    if keys is None:
        keys = _new_keys(st, dev, len(layers), k_new.shape[1], ch)
    bt, kn, kd = desc(block_table), desc(k_new), desc(keys)
    ks = desc(k_scales) if k_scales is not None else None
    check(load().daric_kv_deviation(_layer_array(layers), len(layers), 1 if page_first else 0,
                                    ctypes.byref(bt), ctypes.byref(kn), carr, n,
                                    ctypes.byref(ks) if ks is not None else None, ctypes.byref(kd),
                                    ctypes.c_uint64(st)))
    _record(st, dev, block_table, k_new, keys, k_scales)
    return keys


def topk_per_chunk(keys: torch.Tensor, chunks, kmax: Optional[int] = None,
                   out: Optional[torch.Tensor] = None, stream: int = 0) -> torch.Tensor:
    """Per (layer, chunk) the k largest keys, ties to the lower index; chunk-
    local indices ascending, padded with -1 to kmax."""
    ch = list(chunks)
    if kmax is None:
        kmax = max([min(int(c[3]), int(c[2])) for c in ch] + [0])
    if out is None:
        out = torch.empty(keys.shape[0], len(ch), kmax, dtype=torch.int32, device=keys.device)
    st = _resolve_stream(stream, keys.device)
    carr, n, _keep = _chunks(ch)
    kd, od = desc(keys), desc(out)
    check(load().daric_topk_per_chunk(ctypes.byref(kd), carr, n, ctypes.byref(od), ctypes.c_uint64(st)))
    _record(st, keys.device, keys, out)
    return out


def merge_rows(layers: Sequence[torch.Tensor], page_first: bool, block_table: torch.Tensor,
               k_new: torch.Tensor, v_new: Optional[torch.Tensor], chunks, sel_idx: torch.Tensor,
               stream: int = 0, k_scales: Optional[torch.Tensor] = None,
               v_scales: Optional[torch.Tensor] = None) -> None:
    """Write the selected recomputed K/V rows into their paged-cache slots.
    Rows in the cache's element type are copied; bf16/fp16 rows for an fp8
    (e4m3) cache are quantised as sat_rtne(x / scale) with the [L, H] fp32
    k_scales / v_scales (the fp8 write of vLLM's reshape_and_cache)."""
    layers = list(layers)
    dev = layers[0].device
    st = _resolve_stream(stream, dev)
    carr, n, _keep = _chunks(chunks)
    bt, kn, si = desc(block_table), desc(k_new), desc(sel_idx)
    vn = desc(v_new) if v_new is not None else None
    ks = desc(k_scales) if k_scales is not None else None
    vs = desc(v_scales) if v_scales is not None else None
    check(load().daric_merge_rows(_layer_array(layers), len(layers), 1 if page_first else 0,
                                  ctypes.byref(bt), ctypes.byref(kn),
                                  ctypes.byref(vn) if vn is not None else None, carr, n,
                                  ctypes.byref(si), ctypes.byref(ks) if ks is not None else None,
                                  ctypes.byref(vs) if vs is not None else None, ctypes.c_uint64(st)))
    _record(st, dev, block_table, k_new, v_new, sel_idx, k_scales, v_scales)


SELECT_KEYS_READY = 1       # DARIC_SELECT_KEYS_READY
SELECT_ONE_PASS = 2         # DARIC_SELECT_ONE_PASS


def select_merge(layers: Sequence[torch.Tensor], page_first: bool, block_table: torch.Tensor,
                 k_new: torch.Tensor, v_new: Optional[torch.Tensor], chunks, kmax: Optional[int] = None,
                 keys: Optional[torch.Tensor] = None, sel_idx: Optional[torch.Tensor] = None,
                 keys_ready: bool = False, k_scales: Optional[torch.Tensor] = None,
                 v_scales: Optional[torch.Tensor] = None, stream: int = 0, one_pass: bool = False):
    """kv_deviation + topk_per_chunk + merge_rows in one call: returns
    (keys [L, T] fp32, sel_idx [L, n_chunks, kmax] int32), equal to what the
    three calls return, and merges the selected rows the same way. Where the
    chunks fit, the top-k and merge run fused, one workgroup per (layer,
    chunk). For an fp8 cache, k_scales / v_scales are its [L, H] per-head K / V
    scales. keys_ready: `keys` already holds the deviation keys. one_pass: the
    fused workgroups compute the keys too (one launch; measured slower)."""
    layers = list(layers)
    dev = layers[0].device
    st = _resolve_stream(stream, dev)
    carr, n, ch = _chunks(chunks if isinstance(chunks, np.ndarray) else list(chunks))
    if kmax is None:
        kmax = max(0, int(np.minimum(ch[:, 2], ch[:, 3]).max()))
    if keys is None:
        if keys_ready:
            raise ValueError("keys_ready needs keys")
        keys = _new_keys(st, dev, len(layers), k_new.shape[1], ch)
    if sel_idx is None:
        with _on_stream(st, dev):
            sel_idx = torch.empty(len(layers), n, kmax, dtype=torch.int32, device=dev)
    bt, kn, kd, si = desc(block_table), desc(k_new), desc(keys), desc(sel_idx)
    vn = desc(v_new) if v_new is not None else None
    ks = desc(k_scales) if k_scales is not None else None
    vs = desc(v_scales) if v_scales is not None else None
    check(load().daric_select_merge(_layer_array(layers), len(layers), 1 if page_first else 0,
                                    ctypes.byref(bt), ctypes.byref(kn),
                                    ctypes.byref(vn) if vn is not None else None, carr, n,
                                    ctypes.byref(ks) if ks is not None else None,
                                    ctypes.byref(vs) if vs is not None else None,
                                    ctypes.byref(kd), ctypes.byref(si),
                                    (SELECT_KEYS_READY if keys_ready else 0) | (SELECT_ONE_PASS if one_pass else 0),
                                    ctypes.c_uint64(st)))
    _record(st, dev, block_table, k_new, v_new, keys, sel_idx, k_scales, v_scales)
    return keys, sel_idx


def _tuples(entries, widths, what):
    """(address of int64 [n, widths[0]], n, keep-alive, list of columns) of a
    sequence of integer tuples or an int64 array; entries shorter than
    widths[0] (but of a width named) get zeros behind."""
    full = widths[0]
    a = np.asarray(entries if isinstance(entries, np.ndarray) else list(entries))
    if a.size == 0:
        a = np.zeros((0, full), np.int64)
    if a.ndim != 2 or a.shape[1] not in widths or a.dtype.kind not in "iu":
        raise ValueError(what)
    if a.shape[1] < full:
        a = np.concatenate([a, np.zeros((a.shape[0], full - a.shape[1]), np.int64)], axis=1)
    a = np.ascontiguousarray(a, dtype=np.int64)
    return a.ctypes.data, a.shape[0], a


_SEQUENCES = "sequences must be (bt_offset, row_start, n_rows, n_ctx[, col_start]) entries of ints"


def _sequences(seqs):
    return _tuples(seqs, (5, 4), _SEQUENCES)


_ROW_STRUCTS: dict = {}


def _rows_of_ints(entries, widths, what: str):
    """(int64 [n, widths[0]] as bytes or its address, n, keep-alive) of integer tuples, as
    _tuples, where widths[1], if there is one, is one less. Lists without a Python-level loop
    or numpy: 48 tuples of four ints take 5 us on the host, through numpy 17."""
    if type(entries) is list and entries:
        try:
            n, width = len(entries), len(entries[0])
            if n <= 1024 and width in widths and set(map(len, entries)) == {width}:
                pack = _ROW_STRUCTS.get((n, width, widths))
                if pack is None:
                    if len(_ROW_STRUCTS) >= 256:
                        _ROW_STRUCTS.clear()
                    row = f"{width}q{8 * (widths[0] - width)}x"
                    pack = _ROW_STRUCTS[(n, width, widths)] = struct.Struct("@" + row * n).pack
                return pack(*chain.from_iterable(entries)), n, None
        except (TypeError, struct.error):       # not ints: numpy converts or refuses them
            pass
    return _tuples(entries, widths, what)


def _ref(t: Optional[torch.Tensor]):
    return ctypes.byref(desc(t)) if t is not None else None


def _scale(scale: Optional[float], q: torch.Tensor) -> float:
    """The scores' factor; without one, that of q's head size (the library refuses
    a q that has none)."""
    return float(scale) if scale is not None else q.shape[-1] ** -0.5 if q.dim() and q.shape[-1] else 1.0


def _no_backward(what: str, *tensors) -> None:
    """These calls have no backward pass and carry no forward-mode tangents: an input that
    asks for a gradient, or has a tangent, is refused, not answered by an output that
    silently has none."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad(), or detach what "
                                   "requires a gradient")
    if _in_dual_level():
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what} carries no forward-mode tangents: pass the primal of what has one")


def _layer_desc(layer: torch.Tensor):
    return _layer_array((layer,))


def attend_pages(layer: torch.Tensor, page_first: bool, block_table: torch.Tensor, q: torch.Tensor, seqs,
                 tree_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                 k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                 stream: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of q ([T, Hq, D]) over one layer's paged cache: (out [T, Hq, D]
    of q's type, lse [T, Hq] fp32). seqs: (bt_offset, row_start, n_rows, n_ctx
    [, col_start]); rows row_start .. + n_rows of q belong to tokens that stand in
    the cache behind the sequence's n_ctx cached ones. Every row sees the n_ctx
    tokens; of the others row i sees the first i + 1 (one token, a prompt's run
    of rows), or those whose bits its row of tree_mask (int64 [T, words])
    sets (drafted trees). Tokens in pages of id 0 are not there; rows that see
    nothing get zeros and lse -inf; rows of no sequence are not written. out and
    lse must overlap neither each other nor an input. scale: D ** -0.5 if None. k_scale, v_scale: [H] fp32 scales of an fp8 cache. See
    include/daric_cache_ops.h for what the arguments may be. No backward pass:
    inputs that require a gradient are refused while gradients are enabled."""
    _no_backward("attend_pages", layer, q, k_scale, v_scale, out, lse)
    dev = layer.device
    st = _resolve_stream(stream, dev)
    addr, n, _keep = _sequences(seqs)
    lib, ld, qd = load(), _layer_desc(layer), desc(q)
    pf = 1 if page_first else 0
    need = ctypes.c_int64()
    check(lib.daric_attend_workspace(ld, pf, ctypes.byref(qd), addr, n, ctypes.byref(need)))
    work = None
    if need.value or out is None or lse is None:
        with _on_stream(st, dev):
            if out is None:
                out = torch.empty(q.shape, dtype=q.dtype, device=dev)
            if lse is None:
                lse = torch.empty(q.shape[:2], dtype=torch.float32, device=dev)
            if need.value:
                work = torch.empty(need.value, dtype=torch.uint8, device=dev)
    check(lib.daric_attend_pages(ld, pf, _ref(block_table), ctypes.byref(qd), addr, n, _ref(tree_mask),
                                 _scale(scale, q), _ref(k_scale), _ref(v_scale),
                                 _ref(out), _ref(lse), work.data_ptr() if work is not None else None, need.value,
                                 ctypes.c_uint64(st)))
    _record(st, dev, block_table, q, tree_mask, k_scale, v_scale, out, lse, work)
    return out, lse


def weigh_tokens(layer: torch.Tensor, page_first: bool, block_table: torch.Tensor, q: torch.Tensor,
                 lse: torch.Tensor, seqs, weights: Optional[torch.Tensor] = None,
                 tree_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                 k_scale: Optional[torch.Tensor] = None, stream: int = 0) -> torch.Tensor:
    """The attention weight that each token of the cache received in
    attend_pages(layer, ..., q, seqs, ...), whose lse is passed, summed over the rows
    and the query heads of each KV head: added to weights[:, col_start + j]
    ([H, columns] fp32) for token j of a sequence (bt_offset, row_start, n_rows,
    n_ctx, col_start), or without `weights` written to a new tensor, zeros where
    no sequence is. Returns the weights. No backward pass, as attend_pages."""
    _no_backward("weigh_tokens", layer, q, lse, weights, k_scale)
    dev = layer.device
    st = _resolve_stream(stream, dev)
    addr, n, a = _sequences(seqs)
    fresh = weights is None
    ld, qd = _layer_desc(layer), desc(q)
    if fresh:
        end = int((a[:, 4] + a[:, 2] + a[:, 3]).max()) if n else 0
        heads = layer.shape[1] if layer.dim() == 4 else layer.shape[3] if layer.dim() == 5 else 1
        with _on_stream(st, dev):
            weights = torch.zeros((heads, max(end, 0)), dtype=torch.float32, device=dev)
    check(load().daric_weigh_tokens(ld, 1 if page_first else 0, _ref(block_table), ctypes.byref(qd), _ref(lse), addr, n,
                                    _ref(tree_mask), _scale(scale, q),
                                    _ref(k_scale), _ref(weights), 0 if fresh else 1, ctypes.c_uint64(st)))
    _record(st, dev, block_table, q, lse, tree_mask, k_scale, weights)
    return weights


def evict_tokens(layers: Sequence[torch.Tensor], page_first: bool, block_table: torch.Tensor,
                 weights: torch.Tensor, evictions, stream: int = 0) -> torch.Tensor:
    """Keeps the heaviest tokens of each sequence, per layer and KV head, and
    brings them to its first slots, in place. evictions: (bt_offset, col_start,
    n_tokens, keep, n_first, n_recent); weights: [L, H, columns] fp32 ([L, 1,
    columns]: one choice for all heads of a layer). Kept tokens among the first
    `keep` slots stay, the i-th slot freed takes the i-th kept token from behind.
    Returns kept [L, H or 1, n, kmax] int32: the token that each slot holds
    now, -1 behind the last. The weights move with their tokens, those from
    `keep` on become 0. Rows are bytes: any cache type, MLA caches too. A slot is
    then no longer its position's: not for the calls that pair slots with tokens
    (kv_deviation, merge_rows, select_merge, records of reusable chunks). No
    backward pass, as attend_pages."""
    layers = list(layers)
    _no_backward("evict_tokens", weights, *layers)
    dev = layers[0].device
    st = _resolve_stream(stream, dev)
    addr, n, a = _tuples(evictions, (6,), "evictions must be (bt_offset, col_start, n_tokens, keep, n_first, n_recent) "
                                          "entries of ints")
    kmax = max(0, int(np.minimum(a[:, 2], a[:, 3]).max())) if n else 0
    with _on_stream(st, dev):
        both = torch.empty((2, len(layers), weights.shape[1] if weights.dim() == 3 else 1, n, kmax), dtype=torch.int32,
                           device=dev)
    kept, work = both[0], both[1]
    check(load().daric_evict_tokens(_layer_array(layers), len(layers), 1 if page_first else 0, _ref(block_table),
                                    _ref(weights), addr, n, _ref(kept), _ref(work), ctypes.c_uint64(st)))
    _record(st, dev, block_table, weights, both)
    return kept


def rotate_rows(rows: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, rotary_dim: int,
                is_neox_style: bool = True, attention_scale: float = 1.0, out: Optional[torch.Tensor] = None,
                stream: int = 0) -> torch.Tensor:
    """Rotary positions of new rows ([T, H, D] bf16, fp16 or fp32: queries, keys, or both
    where their heads stand side by side): pair i of the first rotary_dim values
    turns by positions[t] * inv_freq[i] (int64 [T]; angles in fp64), cosine and sine
    times attention_scale; the other values are copied. Pairs are (i, i +
    rotary_dim / 2), or (2i, 2i + 1) with is_neox_style False. out: `rows` itself, or a
    contiguous tensor (made if None). Frequencies of scaled models:
    daric_amd.rotary.rotary_frequencies. Cached rows move by rerotate_pages. No
    backward pass; the gradient of rows is rotate_rows of out's at -positions."""
    _no_backward("rotate_rows", rows, inv_freq, out)
    dev = rows.device
    st = _resolve_stream(stream, dev)
    rope = _rope(inv_freq, rotary_dim, is_neox_style, dev)
    given = out                 # what is made here belongs to `st` already
    if out is None:
        with _on_stream(st, dev) if stream else _HERE:
            out = rows.new_empty(rows.shape)
    (rd, pd, od), _keep = views(rows, positions, out)
    check(load().daric_rotate_rows(rd, pd, ctypes.byref(rope), float(attention_scale), od, st))
    _record(st, dev, rows, positions, inv_freq, given)
    return out


def append_tokens(layer: torch.Tensor, page_first: bool, block_table: torch.Tensor, k: torch.Tensor,
                  v: Optional[torch.Tensor], seqs, inv_freq: Optional[torch.Tensor] = None, rotary_dim: int = 0,
                  is_neox_style: bool = True, positions: Optional[torch.Tensor] = None, attention_scale: float = 1.0,
                  q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
                  k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                  stream: int = 0) -> Optional[torch.Tensor]:
    """Writes the rows of k and v ([T, H, D], strides free) into one layer's paged
    cache, K rotated to its position on the way, and rotates the step's q with it: the
    call before attend_pages, with the same seqs (bt_offset, row_start, n_rows, n_ctx
    [, col_start]): row row_start + i becomes token n_ctx + i of the sequence.
    positions: int64 [T] (None: the token's place, n_ctx + i; after an eviction they
    differ); inv_freq None: nothing is rotated. rotary_dim, is_neox_style,
    attention_scale as in rotate_rows. An fp8 (e4m3) cache takes bf16 or fp16 rows as
    sat_rtne(x / scale) with its [H] fp32 k_scale / v_scale (None: 1). MLA rows (v None)
    whose rotated part stands last: rotate_rows of k[..., -R:] in place, then no inv_freq
    here. Tokens in pages
    of id 0 are not written, nor is anything of rows of no sequence; no slot may be
    written by two rows of a call. Returns
    q_out (q itself, or a contiguous tensor, made if None), or None without q. No
    backward pass, as attend_pages."""
    _no_backward("append_tokens", layer, k, v, q, q_out, inv_freq, k_scale, v_scale)
    dev = layer.device
    st = _resolve_stream(stream, dev)
    addr, n, _keep = _rows_of_ints(seqs, (5, 4), _SEQUENCES)
    rope = _rope(inv_freq, rotary_dim, is_neox_style, dev) if inv_freq is not None else None
    if q is None and q_out is not None:
        raise RuntimeError("q_out needs q")
    given = q_out               # what is made here belongs to `st` already
    if q is not None and q_out is None:
        with _on_stream(st, dev) if stream else _HERE:
            q_out = q.new_empty(q.shape)
    (ld, bt, kd, vd, pd, qd, od, ks, vs), _views = views(layer, block_table, k, v, positions, q, q_out, k_scale, v_scale)
    check(load().daric_append_tokens(ld, 1 if page_first else 0, bt, kd, vd, addr, n, pd,
                                     ctypes.byref(rope) if rope is not None else None, float(attention_scale), qd, od,
                                     ks, vs, st))
    _record(st, dev, block_table, k, v, positions, inv_freq, q, given, k_scale, v_scale)
    return q_out


def select_beams(logits: torch.Tensor, scores: torch.Tensor, k: Optional[int] = None,
                 ended: Optional[torch.Tensor] = None, end_token: int = -1,
                 stream: int = 0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The k best continuations (W if None, at most 64) of each request's W beams:
    (scores [B, k] fp32, parents [B, k] int32, tokens [B, k] int32), best first. A
    candidate's score is scores[b, w] + log_softmax(logits[b, w])[v] (logits: [B, W, V]
    bf16, fp16 or fp32; scores: fp32), compared in 64 bits, ties to the lower beam,
    then the larger logit, then the lower token. Beams that `ended` (bool [B, W]) offer
    end_token alone, at their own score. Candidates of score -inf or NaN are not there:
    score -inf, parent and token -1 fill the places left. A beam's log-sum is off by up to
    2.3e-6 (its sums are fp32): closer candidates of different beams may come in either
    order. Up to 64 beams of a request; reorder_beams takes 32. No backward pass, as
    attend_pages."""
    _no_backward("select_beams", logits, scores)
    dev = logits.device
    st = _resolve_stream(stream, dev)
    if k is None:
        k = logits.shape[1] if logits.dim() == 3 else 1
    k = int(k)
    shape = (logits.shape[0] if logits.dim() else 0, k)
    with _on_stream(st, dev) if stream else _HERE:
        out = torch.empty(shape, dtype=torch.float32, device=dev)
        parents = torch.empty(shape, dtype=torch.int32, device=dev)
        tokens = torch.empty(shape, dtype=torch.int32, device=dev)
    end = ended.view(torch.uint8) if ended is not None and ended.dtype == torch.bool else ended
    (ld, sd, ed, od, pd, td), _views = views(logits, scores, end, out, parents, tokens)
    lib, need = load(), ctypes.c_int64()
    check(lib.daric_select_workspace(ld, k, ctypes.byref(need)))
    with _on_stream(st, dev) if stream else _HERE:
        work = torch.empty(need.value, dtype=torch.uint8, device=dev)
    check(lib.daric_select_beams(ld, sd, ed, int(end_token), od, pd, td, work.data_ptr(), need.value, st))
    _record(st, dev, logits, scores, end)
    return out, parents, tokens


def reorder_beams(layers: Sequence[torch.Tensor], page_first: bool, block_table: torch.Tensor,
                  parents: torch.Tensor, beams, stream: int = 0) -> None:
    """Beam w of request i goes on from beam parents[i, w] (int32 [n, columns], -1: it
    stays), in place and without the host: beams holds (bt_offset, stride, n_beams,
    n_tokens) per request, beam w's block list beginning at block_table[bt_offset +
    w * stride]. The ids of its full pages become its parent's, and its last, partly
    filled page, which no other list may hold there, takes the rows of the parent's, in
    every layer at once. Up to 32 beams of a request; caches of any type and
    layout, no two of which share memory."""
    layers = list(layers)
    if _in_dual_level() or (torch.is_grad_enabled() and any(map(_REQUIRES_GRAD, layers))):
        _no_backward("reorder_beams", *layers)
    dev = layers[0].device
    st = _resolve_stream(stream, dev)
    addr, n, _keep = _rows_of_ints(beams, (4,), "beams must be (bt_offset, stride, n_beams, n_tokens) entries of ints")
    (bt, pd), _views = views(block_table, parents)
    check(load().daric_reorder_beams(layer_views(layers), len(layers), 1 if page_first else 0, bt, pd, addr, n, st))
    _record(st, dev, block_table, parents)


def timing_enable(enable: bool = True) -> None:
    check(load().daric_timing_enable(1 if enable else 0))


def timing_read() -> tuple[float, int]:
    """(summed kernel milliseconds, launches) since the last read."""
    ms = ctypes.c_double()
    n = ctypes.c_int64()
    check(load().daric_timing_read(ctypes.byref(ms), ctypes.byref(n)))
    return ms.value, n.value
