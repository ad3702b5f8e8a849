"""Torch-facing wrappers of the C ABI: the reference's kernel entry points.

Mirrors, with the same argument meaning:
  kivi_compressed_bytes / kivi_params_supported / kivi_compress / kivi_decompress
      src/inference/backends/cuda/compression/kivi_cache.cuh:32-84
  reshape_and_cache  -> paged_append    (cuda_engine.cpp:48-50, cache_kernels.cu:202-232)
  paged_attention_v1/v2 -> paged_decode (cuda_engine.cpp:51-62)
and, beside the KIVI cache, the paged int8 cache (int8_append, int8_read,
int8_attend) and rotary positions with several axes (rope_axes).
Every call goes to the sm_100a library; tensors must be CUDA tensors.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
from dataclasses import dataclass
from typing import Optional

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _lib as L

_DT = {torch.float16: L.TKV_F16, torch.bfloat16: L.TKV_BF16, torch.float32: L.TKV_F32}


def _stream(stream) -> int:
    if stream is None:
        return torch.cuda.current_stream().cuda_stream
    if isinstance(stream, torch.cuda.Stream):
        return stream.cuda_stream
    return int(stream)


def _ptr(t: Optional[torch.Tensor]):
    if t is None:
        return None
    return C.c_void_p(t.data_ptr())


def _need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("KIVI kernels take CUDA tensors")


# ---------------------------------------------------------------------------
# reference-format KIVI (kivi_cache.cuh)
# ---------------------------------------------------------------------------
KIVI_MAX_HEAD_DIM = 128  # kivi_cache.cuh:27
KIVI_MAX_OUTLIERS = 64  # kivi_cache.cuh:28


def kivi_compressed_bytes(head_dim: int, n_outliers: int, group_size: int) -> int:
    """Bytes of one compressed vector (kivi_cache.cuh:32-43)."""
    return int(L.lib().tkv_kivi_compressed_bytes(head_dim, n_outliers, group_size))


def kivi_params_supported(head_dim: int, n_outliers: int, group_size: int) -> bool:
    """kivi_cache.cu:205-211."""
    return bool(L.lib().tkv_kivi_params_supported(head_dim, n_outliers, group_size))


def kivi_compress(d_kv_in: torch.Tensor, d_out: torch.Tensor, n_vecs: int, head_dim: int,
                  n_outliers: int, group_size: int, stream=None) -> None:
    """truellm::kivi_compress: a no-op when kivi_params_supported() is false or
    n_vecs <= 0, as in the reference wrapper (kivi_cache.cu:213-225)."""
    if n_vecs <= 0 or not kivi_params_supported(head_dim, n_outliers, group_size):
        return
    _need_cuda(d_kv_in, d_out)
    L.check("tkv_kivi_compress", L.lib().tkv_kivi_compress(
        _ptr(d_kv_in), _ptr(d_out), n_vecs, head_dim, n_outliers, group_size,
        C.c_void_p(_stream(stream))))


def kivi_decompress(d_in: torch.Tensor, d_kv_out: torch.Tensor, n_vecs: int, head_dim: int,
                    n_outliers: int, group_size: int, stream=None) -> None:
    """truellm::kivi_decompress (kivi_cache.cu:227-239)."""
    if n_vecs <= 0 or not kivi_params_supported(head_dim, n_outliers, group_size):
        return
    _need_cuda(d_in, d_kv_out)
    L.check("tkv_kivi_decompress", L.lib().tkv_kivi_decompress(
        _ptr(d_in), _ptr(d_kv_out), n_vecs, head_dim, n_outliers, group_size,
        C.c_void_p(_stream(stream))))


def kivi_roundtrip_inplace(d_kv: torch.Tensor, n_vecs: int, head_dim: int, n_outliers: int,
                           group_size: int, stream=None) -> None:
    """compress + decompress in place in one launch (KvCompressionPass::run_kivi)."""
    if n_vecs <= 0 or not kivi_params_supported(head_dim, n_outliers, group_size):
        return
    _need_cuda(d_kv)
    L.check("tkv_kivi_roundtrip_inplace", L.lib().tkv_kivi_roundtrip_inplace(
        _ptr(d_kv), n_vecs, head_dim, n_outliers, group_size, C.c_void_p(_stream(stream))))


# ---------------------------------------------------------------------------
# paged KIVI cache
# ---------------------------------------------------------------------------
@dataclass(frozen=True)
class KiviFormat:
    head_dim: int
    group_size: int
    residual: int
    bits: int
    n_kv_heads: int

    def c_struct(self) -> L.TkvFormat:
        f = L.TkvFormat()
        L.check("tkv_format_init", L.lib().tkv_format_init(
            C.byref(f), self.head_dim, self.group_size, self.residual, self.bits,
            self.n_kv_heads))
        return f

    @property
    def page_bytes(self) -> int:
        return int(self.c_struct().page_bytes)

    @property
    def ring_cap(self) -> int:
        return int(self.c_struct().ring_cap)

    def quantized_len(self, length: int) -> int:
        x = length - self.residual
        return self.group_size * (x // self.group_size) if x > 0 else 0


class KiviPagedCache:
    """Device buffers of one layer's paged KIVI cache.

    pool: [num_pages, n_kv_heads, page_bytes] uint8 (block-major like the
    reference pool, cuda_allocator.h:9-12); ring: [max_seqs, n_kv_heads,
    ring_cap/16, 2, 16*D] fp16 residual window.  Both zero-initialised.
    """

    def __init__(self, fmt: KiviFormat, num_pages: int, max_seqs: int, device="cuda"):
        self.fmt = fmt
        cf = fmt.c_struct()
        self.num_pages = int(num_pages)
        self.max_seqs = int(max_seqs)
        self.pool = torch.zeros((num_pages, fmt.n_kv_heads, int(cf.page_bytes)),
                                dtype=torch.uint8, device=device)
        self.ring = torch.zeros((max_seqs, fmt.n_kv_heads, int(cf.ring_cap) // 16, 2,
                                 16 * fmt.head_dim), dtype=torch.float16, device=device)

    def c_struct(self) -> L.TkvCache:
        c = L.TkvCache()
        c.pool = self.pool.data_ptr()
        c.ring = self.ring.data_ptr()
        c.num_pages = self.num_pages
        c.max_seqs = self.max_seqs
        c.fmt = self.fmt.c_struct()
        return c


def paged_append(cache: KiviPagedCache, k_new: torch.Tensor, v_new: torch.Tensor,
                 cu_new: torch.Tensor, seq_lens_old: torch.Tensor, block_tables: torch.Tensor,
                 seq_slots: Optional[torch.Tensor] = None, max_new_tokens: Optional[int] = None,
                 err: Optional[torch.Tensor] = None, stream=None) -> None:
    """Quantize-on-append (the KIVI reshape_and_cache).

    k_new, v_new: [T_total, n_kv_heads, D] fp16/bf16; cu_new: [B+1] int32 token
    offsets; seq_lens_old: [B] int32; block_tables: [B, max_blocks] int32.
    max_new_tokens bounds the per-sequence token count (defaults to T_total).
    """
    _need_cuda(k_new, v_new, cu_new, seq_lens_old, block_tables)
    if k_new.dtype not in (torch.float16, torch.bfloat16) or v_new.dtype != k_new.dtype:
        raise ValueError("k_new/v_new must both be fp16 or bf16")
    B = int(seq_lens_old.numel())
    mnt = int(k_new.shape[0]) if max_new_tokens is None else int(max_new_tokens)
    c = cache.c_struct()
    L.check("tkv_paged_append", L.lib().tkv_paged_append(
        C.byref(c), _ptr(k_new.contiguous()), _ptr(v_new.contiguous()), _DT[k_new.dtype],
        _ptr(cu_new), _ptr(seq_lens_old), _ptr(block_tables), int(block_tables.shape[1]),
        _ptr(seq_slots), B, int(k_new.shape[0]), mnt, _ptr(err), C.c_void_p(_stream(stream))))


def decode_workspace_bytes(num_seqs: int, num_q_heads: int, head_dim: int,
                           max_context_len: int) -> int:
    return int(L.lib().tkv_decode_workspace_bytes(num_seqs, num_q_heads, head_dim,
                                                  max_context_len))


def decode_range_workspace_bytes(num_seqs: int, num_q_heads: int, head_dim: int,
                                 split_lo: int, split_hi: int) -> int:
    return int(L.lib().tkv_decode_range_workspace_bytes(num_seqs, num_q_heads, head_dim,
                                                        split_lo, split_hi))


def decode_launches(num_seqs: int, num_q_heads: int, num_kv_heads: int,
                    max_context_len: int) -> int:
    """Kernel launches one paged_decode call makes on the current device: 1
    (merge fused into the decode kernel), or 2 when there is less than one
    (sequence, kv head) pair per 16 resident warps (a separate merge kernel
    spreads the merge of pairs that span many warps over the GPU)."""
    return int(L.lib().tkv_decode_launches(num_seqs, num_q_heads, num_kv_heads,
                                           max_context_len))


def decode_num_splits(max_context_len: int) -> int:
    return int(L.lib().tkv_decode_num_splits(max_context_len))


def paged_decode(cache: KiviPagedCache, q: torch.Tensor, block_tables: torch.Tensor,
                 seq_lens: torch.Tensor, max_context_len: int, scale: Optional[float] = None,
                 out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                 workspace: Optional[torch.Tensor] = None,
                 seq_slots: Optional[torch.Tensor] = None, err: Optional[torch.Tensor] = None,
                 stream=None) -> torch.Tensor:
    """Decode attention over the KIVI cache (the paged_attention_v1/v2 slot).

    q: [B, Hq, D] fp16/bf16.  Returns out [B, Hq, D] (dtype of q unless
    out/out_dtype say otherwise).  scale defaults to 1/sqrt(D) (cuda_engine.cpp:1140).
    """
    _need_cuda(q, block_tables, seq_lens)
    B, Hq, D = q.shape
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty((B, Hq, D), dtype=out_dtype or q.dtype, device=q.device)
    ws_bytes = decode_workspace_bytes(B, Hq, D, max_context_len)
    if workspace is None:  # work counters at its start must be zero: allocate zeroed
        workspace = torch.zeros(ws_bytes, dtype=torch.uint8, device=q.device)
    c = cache.c_struct()
    L.check("tkv_paged_decode", L.lib().tkv_paged_decode(
        C.byref(c), _ptr(q.contiguous()), _DT[q.dtype], _ptr(out), _DT[out.dtype],
        _ptr(block_tables), int(block_tables.shape[1]), _ptr(seq_lens), _ptr(seq_slots), B, Hq,
        float(scale), int(max_context_len), _ptr(workspace), int(workspace.numel()),
        _ptr(err), C.c_void_p(_stream(stream))))
    return out


class PreparedDecode:
    """tkv_paged_decode with its arguments bound once to fixed buffers: each
    call is one ctypes call, for decode loops where the wrapper's per-call
    work (argument conversion, the format struct) would show beside a
    ~0.1 ms kernel.  The buffers must stay alive and keep their addresses."""

    def __init__(self, cache: KiviPagedCache, q: torch.Tensor, block_tables: torch.Tensor,
                 seq_lens: torch.Tensor, max_context_len: int, out: torch.Tensor,
                 workspace: torch.Tensor, scale: Optional[float] = None,
                 seq_slots: Optional[torch.Tensor] = None, err: Optional[torch.Tensor] = None,
                 stream=None):
        _need_cuda(q, block_tables, seq_lens, out, workspace)
        if not q.is_contiguous():
            raise ValueError("q must be contiguous")
        B, Hq, D = q.shape
        if scale is None:
            scale = 1.0 / math.sqrt(D)
        self._keep = (q, block_tables, seq_lens, out, workspace, seq_slots, err)
        self._c = cache.c_struct()
        self._fn = L.lib().tkv_paged_decode
        self._args = (C.byref(self._c), _ptr(q), _DT[q.dtype], _ptr(out), _DT[out.dtype],
                      _ptr(block_tables), int(block_tables.shape[1]), _ptr(seq_lens),
                      _ptr(seq_slots), B, Hq, float(scale), int(max_context_len),
                      _ptr(workspace), int(workspace.numel() * workspace.element_size()),
                      _ptr(err), C.c_void_p(_stream(stream)))

    def __call__(self) -> None:
        st = self._fn(*self._args)
        if st != L.TKV_OK:
            raise L.TkvError("tkv_paged_decode", st)


def paged_decode_partials(cache: KiviPagedCache, q: torch.Tensor, block_tables: torch.Tensor,
                          seq_lens: torch.Tensor, split_lo: int, split_hi: int,
                          include_residual: bool, part_ml: torch.Tensor, part_o: torch.Tensor,
                          scale: Optional[float] = None,
                          seq_slots: Optional[torch.Tensor] = None,
                          err: Optional[torch.Tensor] = None,
                          work: Optional[torch.Tensor] = None, stream=None) -> None:
    """Split-KV partials (m, l, o) of quantised splits [split_lo, split_hi)
    (+ the residual split) for sequences split across GPUs.  work: >= 8 bytes
    of zeroed device memory reused across calls (allocated when omitted)."""
    _need_cuda(q, block_tables, seq_lens, part_ml, part_o)
    if work is None:
        work = torch.zeros(2, dtype=torch.int32, device=q.device)
    B, Hq, D = q.shape
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    c = cache.c_struct()
    L.check("tkv_paged_decode_partials", L.lib().tkv_paged_decode_partials(
        C.byref(c), _ptr(q.contiguous()), _DT[q.dtype], _ptr(block_tables),
        int(block_tables.shape[1]), _ptr(seq_lens), _ptr(seq_slots), B, Hq, float(scale),
        int(split_lo), int(split_hi), int(bool(include_residual)), _ptr(part_ml), _ptr(part_o),
        _ptr(work), _ptr(err), C.c_void_p(_stream(stream))))


def paged_decode_range(cache: KiviPagedCache, q: torch.Tensor, block_tables: torch.Tensor,
                       seq_lens: torch.Tensor, split_lo: int, split_hi: int,
                       include_residual: bool, out_ml: torch.Tensor, out_o: torch.Tensor,
                       workspace: torch.Tensor, scale: Optional[float] = None,
                       seq_slots: Optional[torch.Tensor] = None,
                       err: Optional[torch.Tensor] = None, stream=None) -> None:
    """One GPU's share of a token-split decode: quantised splits [split_lo,
    split_hi) (+ the residual split) reduced in the launch to one partial per
    (sequence, q head): out_ml [B, Hq, 2], out_o [B, Hq, D] fp32.  workspace:
    zeroed uint8 device tensor of decode_range_workspace_bytes(B, Hq, D,
    split_lo, split_hi) bytes, reused across calls."""
    _need_cuda(q, block_tables, seq_lens, out_ml, out_o, workspace)
    B, Hq, D = q.shape
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    c = cache.c_struct()
    L.check("tkv_paged_decode_range", L.lib().tkv_paged_decode_range(
        C.byref(c), _ptr(q.contiguous()), _DT[q.dtype], _ptr(block_tables),
        int(block_tables.shape[1]), _ptr(seq_lens), _ptr(seq_slots), B, Hq, float(scale),
        int(split_lo), int(split_hi), int(bool(include_residual)), _ptr(out_ml), _ptr(out_o),
        _ptr(workspace), int(workspace.numel() * workspace.element_size()), _ptr(err),
        C.c_void_p(_stream(stream))))


def paged_prefill(cache: KiviPagedCache, q: torch.Tensor, cu_q: torch.Tensor,
                  block_tables: torch.Tensor, seq_lens: torch.Tensor,
                  max_q_tokens: Optional[int] = None, scale: Optional[float] = None,
                  out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                  seq_slots: Optional[torch.Tensor] = None, err: Optional[torch.Tensor] = None,
                  stream=None) -> torch.Tensor:
    """Causal chunked-prefill attention over the KIVI cache: q [T, Hq, D]
    holds, per sequence, its last cu_q[s+1]-cu_q[s] tokens (already appended);
    seq_lens are the lengths after the append.  Returns out [T, Hq, D]."""
    _need_cuda(q, cu_q, block_tables, seq_lens)
    T, Hq, D = q.shape
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty((T, Hq, D), dtype=out_dtype or q.dtype, device=q.device)
    mq = T if max_q_tokens is None else int(max_q_tokens)
    c = cache.c_struct()
    L.check("tkv_paged_prefill", L.lib().tkv_paged_prefill(
        C.byref(c), _ptr(q.contiguous()), _DT[q.dtype], _ptr(out), _DT[out.dtype], _ptr(cu_q),
        _ptr(block_tables), int(block_tables.shape[1]), _ptr(seq_lens), _ptr(seq_slots),
        int(seq_lens.numel()), Hq, T, mq, float(scale), _ptr(err), C.c_void_p(_stream(stream))))
    return out


def merge_partials(part_ml: torch.Tensor, part_o: torch.Tensor, out: torch.Tensor,
                   stream=None) -> torch.Tensor:
    """LSE merge (paged_attention_v2.cu:132-170).  part_ml: [S, B, Hq, 2],
    part_o: [S, B, Hq, D] fp32; out: [B, Hq, D]."""
    _need_cuda(part_ml, part_o, out)
    S, B, Hq, D = part_o.shape
    L.check("tkv_merge_partials", L.lib().tkv_merge_partials(
        _ptr(part_ml), _ptr(part_o), S, B, Hq, D, _ptr(out), _DT[out.dtype],
        C.c_void_p(_stream(stream))))
    return out


# ---------------------------------------------------------------------------
# token split over peer memory (tkv_exchange_*)
# ---------------------------------------------------------------------------
def exchange_buffer_bytes(world: int, num_seqs: int, num_q_heads: int, head_dim: int) -> int:
    return int(L.lib().tkv_exchange_buffer_bytes(world, num_seqs, num_q_heads, head_dim))


class DeviceBuffer:
    """Zeroed device memory from tkv_device_alloc (shareable over CUDA IPC) on
    the current device; freed by close()."""

    def __init__(self, nbytes: int):
        p = C.c_void_p()
        L.check("tkv_device_alloc", L.lib().tkv_device_alloc(int(nbytes), C.byref(p)))
        self.ptr, self.nbytes = int(p.value), int(nbytes)

    def close(self) -> None:
        if self.ptr:
            L.check("tkv_device_free", L.lib().tkv_device_free(C.c_void_p(self.ptr)))
            self.ptr = 0


def ipc_handle(ptr: int) -> bytes:
    h = (C.c_char * L.TKV_IPC_HANDLE_BYTES)()
    L.check("tkv_ipc_get_handle", L.lib().tkv_ipc_get_handle(C.c_void_p(ptr), h))
    return bytes(h)


def ipc_open(handle: bytes) -> int:
    h = (C.c_char * L.TKV_IPC_HANDLE_BYTES).from_buffer_copy(handle)
    p = C.c_void_p()
    L.check("tkv_ipc_open_handle", L.lib().tkv_ipc_open_handle(h, C.byref(p)))
    return int(p.value)


def ipc_close(ptr: int) -> None:
    L.check("tkv_ipc_close_handle", L.lib().tkv_ipc_close_handle(C.c_void_p(ptr)))


def exchange_struct(world: int, rank: int, buffers) -> L.TkvExchange:
    ex = L.TkvExchange()
    ex.world, ex.rank = int(world), int(rank)
    for r, b in enumerate(buffers):
        ex.buffers[r] = int(b)
    return ex


def exchange_decode_range(cache: KiviPagedCache, q: torch.Tensor, block_tables: torch.Tensor,
                          seq_lens: torch.Tensor, split_lo: int, split_hi: int,
                          include_residual: bool, ex: L.TkvExchange,
                          workspace: Optional[torch.Tensor], scale: Optional[float] = None,
                          seq_slots: Optional[torch.Tensor] = None,
                          err: Optional[torch.Tensor] = None, stream=None) -> None:
    """This GPU's range of a token split (see paged_decode_range), reduced and
    stored into every GPU's exchange buffer, flag raised."""
    _need_cuda(q, block_tables, seq_lens)
    B, Hq, D = q.shape
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    c = cache.c_struct()
    ws_bytes = 0 if workspace is None else int(workspace.numel() * workspace.element_size())
    L.check("tkv_exchange_decode_range", L.lib().tkv_exchange_decode_range(
        C.byref(c), _ptr(q.contiguous()), _DT[q.dtype], _ptr(block_tables),
        int(block_tables.shape[1]), _ptr(seq_lens), _ptr(seq_slots), B, Hq, float(scale),
        int(split_lo), int(split_hi), int(bool(include_residual)), C.byref(ex), _ptr(workspace),
        ws_bytes, _ptr(err), C.c_void_p(_stream(stream))))


def exchange_merge(ex: L.TkvExchange, out: torch.Tensor, err: Optional[torch.Tensor] = None,
                   stream=None) -> torch.Tensor:
    """Waits for every GPU's partials of this step and merges them into out
    [B, Hq, D] (f32, f16 or bf16)."""
    _need_cuda(out)
    B, Hq, D = out.shape
    L.check("tkv_exchange_merge", L.lib().tkv_exchange_merge(
        C.byref(ex), B, Hq, D, _ptr(out), _DT[out.dtype], _ptr(err), C.c_void_p(_stream(stream))))
    return out


# ---------------------------------------------------------------------------
# page and ring-row moves (copy_blocks / swap_blocks, cache_kernels.cu:107-168)
# ---------------------------------------------------------------------------
def _mapping(mapping: torch.Tensor) -> int:
    if mapping.dtype != torch.int32 or mapping.dim() != 2 or mapping.shape[1] != 2:
        raise ValueError("mapping must be an int32 [n, 2] tensor of (src, dst) pairs")
    if not (mapping.is_cuda or mapping.is_pinned()):
        raise ValueError("mapping must be a CUDA or pinned host tensor")
    return int(mapping.shape[0])


def _images(images: torch.Tensor, like: torch.Tensor) -> None:
    """images must be [capacity, *like.shape[1:]] of like's dtype, contiguous,
    in CUDA or pinned host memory: the kernel addresses whole rows of it."""
    if not (images.is_cuda or images.is_pinned()) or not images.is_contiguous():
        raise ValueError("images must be a contiguous CUDA or pinned host tensor")
    if images.dtype != like.dtype or tuple(images.shape[1:]) != tuple(like.shape[1:]):
        raise ValueError(f"images must be [capacity, {', '.join(map(str, like.shape[1:]))}] "
                         f"{like.dtype}")


def copy_pages(cache: KiviPagedCache, mapping: torch.Tensor, err: Optional[torch.Tensor] = None,
               stream=None) -> None:
    """copy_blocks for KIVI pages: pool page mapping[i,0] -> mapping[i,1]."""
    n = _mapping(mapping)
    c = cache.c_struct()
    L.check("tkv_copy_pages", L.lib().tkv_copy_pages(
        C.byref(c), _ptr(mapping), n, _ptr(err), C.c_void_p(_stream(stream))))


def swap_pages(cache: KiviPagedCache, images: torch.Tensor, mapping: torch.Tensor,
               direction: int, err: Optional[torch.Tensor] = None, stream=None) -> None:
    """swap_blocks for KIVI pages.  images: [capacity, n_kv_heads, page_bytes]
    uint8, pinned host (or CUDA); direction 0 = pool -> images, 1 = images -> pool."""
    n = _mapping(mapping)
    _images(images, cache.pool)
    c = cache.c_struct()
    cap = int(images.shape[0])
    L.check("tkv_swap_pages", L.lib().tkv_swap_pages(
        C.byref(c), _ptr(images), cap, _ptr(mapping), n, int(direction), _ptr(err),
        C.c_void_p(_stream(stream))))


def copy_ring_rows(cache: KiviPagedCache, mapping: torch.Tensor,
                   err: Optional[torch.Tensor] = None, stream=None) -> None:
    """Ring row mapping[i,0] -> mapping[i,1] (the device half of a fork)."""
    n = _mapping(mapping)
    c = cache.c_struct()
    L.check("tkv_copy_ring_rows", L.lib().tkv_copy_ring_rows(
        C.byref(c), _ptr(mapping), n, _ptr(err), C.c_void_p(_stream(stream))))


def swap_ring_rows(cache: KiviPagedCache, images: torch.Tensor, mapping: torch.Tensor,
                   direction: int, err: Optional[torch.Tensor] = None, stream=None) -> None:
    """Ring rows to / from images [capacity, *ring row shape] fp16 (pinned host or CUDA)."""
    n = _mapping(mapping)
    _images(images, cache.ring)
    c = cache.c_struct()
    L.check("tkv_swap_ring_rows", L.lib().tkv_swap_ring_rows(
        C.byref(c), _ptr(images), int(images.shape[0]), _ptr(mapping), n, int(direction),
        _ptr(err), C.c_void_p(_stream(stream))))


# ---------------------------------------------------------------------------
# rotary positions with several axes, and the paged int8 cache
# ---------------------------------------------------------------------------
class _On:
    """Makes a device and the call's stream current, so that what a call
    allocates or copies belongs to the stream its kernel runs on."""

    def __init__(self, index: int, stream):
        device = torch.device("cuda", index)
        if stream is not None and not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(int(stream), device=device)
        if stream is not None and stream.device != device:
            raise ValueError(f"stream is on {stream.device}, the tensors on {device}")
        self._ctx = [torch.cuda.device(device)]
        if stream is not None:
            self._ctx.append(torch.cuda.stream(stream))
        self._index = index

    def __enter__(self) -> int:
        for c in self._ctx:
            c.__enter__()
        return torch.cuda.current_stream(self._index).cuda_stream

    def __exit__(self, *exc):
        for c in reversed(self._ctx):
            c.__exit__(*exc)


class _Here:
    """_On's short form for the current device and its current stream: a call on
    one token costs as much on the host as on the GPU."""

    def __init__(self, stream: int):
        self._stream = stream

    def __enter__(self) -> int:
        return self._stream

    def __exit__(self, *exc):
        pass


def _on(index: int, stream):
    if stream is None and torch.cuda.current_device() == index:
        return _Here(torch._C._cuda_getCurrentRawStream(index))
    return _On(index, stream)


def _one_device(index: int, *ts) -> None:
    for t in ts:
        if t is not None and t.get_device() != index:
            if not t.is_cuda:
                raise ValueError("the kernels take CUDA tensors")
            raise ValueError(f"tensors are on devices {t.get_device()} and {index}: one is needed")


def _index(name: str, t: torch.Tensor, shape: tuple) -> int:
    """Address of a contiguous int32 tensor of this shape."""
    if t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 {list(shape)} tensor")
    return t.data_ptr()


def _table(t: torch.Tensor, num_seqs: int) -> tuple:
    """Address and width of a block table."""
    if t.dim() != 2:
        raise ValueError("block_tables must be an int32 [sequences, blocks] tensor")
    n = t.shape[1]
    return _index("block_tables", t, (num_seqs, n)), n


def _count(t: torch.Tensor) -> int:
    return t.shape[0] if t.dim() == 1 else -1


def _i32(name: str, n) -> int:
    """n, which the library takes in 32 bits (ctypes would drop the others)."""
    n = int(n)
    if not -2 ** 31 <= n < 2 ** 31:
        raise ValueError(f"{name} is {n}: 32 bits are supported")
    return n


def _err_ptr(err: Optional[torch.Tensor]):
    if err is None:
        return None
    if err.dtype is not torch.int32 or err.numel() < 1:
        raise ValueError("err must be an int32 tensor of one word")
    return err.data_ptr()


_HALF = (torch.float16, torch.bfloat16)


def _heads(name: str, t: torch.Tensor) -> torch.Tensor:
    """[T, H, D] fp16/bf16 whose 16-byte vectors the kernels can address: any
    token and head strides that are multiples of 8 elements, else a copy."""
    if t.dim() != 3 or t.dtype not in _HALF:
        raise ValueError(f"{name} must be an fp16 or bf16 [tokens, heads, channels] tensor")
    st, sh, sd = t.stride()
    if sd != 1 or (st | sh) & 7 or t.data_ptr() & 15:
        # (contiguous() would keep the strides of an axis of one, and the address)
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _like(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """A new contiguous tensor of x's shape."""
    if x.dtype is dtype and x.is_contiguous():
        return torch.empty_like(x)  # half the host's time of torch.empty
    return torch.empty(x.shape, dtype=dtype, device=x.device)


def _rows(t: torch.Tensor) -> tuple:
    """Of a [tokens, heads, channels] tensor, in bytes: where it starts and ends, its
    outer stride, and what one step along the outer axis spans."""
    (T, H, D), (st, sh, _) = t.shape, t.stride()
    st, sh, size = st if T > 1 else 0, sh if H > 1 else 0, t.element_size()
    row = D + (sh * (H - 1) if st >= sh else st * (T - 1))
    whole = D + st * (T - 1) + sh * (H - 1)
    return t.data_ptr(), t.data_ptr() + size * whole, size * max(st, sh), size * row


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Two tensors lie one after the other, or side by side in rows of one length
    (slices of a fused projection)."""
    a0, a1, a_step, a_row = _rows(a)
    b0, b1, b_step, b_row = _rows(b)
    if a1 <= b0 or b1 <= a0 or not a.numel() or not b.numel():
        return True
    return a_step == b_step > 0 and a_row <= (b0 - a0) % a_step <= a_step - b_row


def _same(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and a.stride() == b.stride()


def _plain(name: str, t: Optional[torch.Tensor]) -> None:
    if t is not None and _differentiated(t):
        raise ValueError(f"{name} requires a gradient or carries a tangent: give a plain tensor")


def _rope_outputs(q, k, q_out, k_out) -> None:
    """Refuses outputs whose elements, or whose and an input's, share memory (they may
    be their inputs)."""
    for name, o, own, other in (("q_out", q_out, q, k), ("k_out", k_out, k, q)):
        if o is None:
            continue
        _plain(name, o)
        (T, H, D), (st, sh, _) = o.shape, o.stride()
        # (of two axes, one steps over all of the other)
        if (T > 1 and st < D or H > 1 and sh < D or
                T > 1 and H > 1 and st < D + sh * (H - 1) and sh < D + st * (T - 1)):
            raise ValueError(f"elements of {name} share memory")
        if not (_same(o, own) or _apart(o, own)) or other is not None and not _apart(o, other):
            raise ValueError(f"{name} overlaps an input")
    if q_out is not None and k_out is not None and not _apart(q_out, k_out):
        raise ValueError("q_out overlaps k_out")


def _written(*outs) -> None:
    """Tells autograd that these were written (a backward pass that needs what they held
    before is then an error)."""
    for t in outs:
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)


_I64x2, _I64x4, _I64x8 = C.c_int64 * 2, C.c_int64 * 4, C.c_int64 * 8


def _differentiated(*ts) -> bool:
    """A gradient or a tangent of some tensor is wanted."""
    grad = torch.is_grad_enabled()
    for t in ts:
        if t is not None and (grad and t.requires_grad or unpack_dual(t)[1] is not None):
            return True
    return False


def _no_grad_path(name: str, *ts) -> None:
    if _differentiated(*ts):
        raise ValueError(f"{name} has no gradient: call it under torch.no_grad(), on tensors "
                         "without tangents")


@functools.lru_cache(maxsize=64)
def _rope_plan(rotary_dim: int, sections: tuple, theta: float, order: str,
               pairing: str) -> L.TkvRopePlan:
    orders = {"blocks": L.TKV_ROPE_BLOCKS, "round_robin": L.TKV_ROPE_ROUND_ROBIN}
    pairings = {"halves": L.TKV_ROPE_HALVES, "adjacent": L.TKV_ROPE_ADJACENT}
    if order not in orders or pairing not in pairings:
        raise ValueError("order is 'blocks' or 'round_robin', pairing 'halves' or 'adjacent'")
    if not 1 <= len(sections) <= L.TKV_ROPE_MAX_AXES:
        raise ValueError(f"1 to {L.TKV_ROPE_MAX_AXES} axes are supported")
    p = L.TkvRopePlan()
    pairs = [_i32("a section", n) for n in sections]
    L.check("tkv_rope_plan_init", L.lib().tkv_rope_plan_init(
        C.byref(p), _i32("rotary_dim", rotary_dim), theta, (C.c_int32 * len(pairs))(*pairs),
        len(pairs), orders[order], pairings[pairing]))
    return p


def rope_axes(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, sections,
              theta: float = 10000.0, order: str = "blocks", pairing: str = "halves",
              inverse: bool = False, q_out: Optional[torch.Tensor] = None,
              k_out: Optional[torch.Tensor] = None, stream=None):
    """Rotary positions with several axes on queries and keys.

    q: [T, Hq, D], k: [T, Hk, D] (or None), both fp16 or both bf16; positions:
    int32 [axes, T]; sections: frequency pairs of each axis, their sum half of
    the rotary channels (channels from 2 * sum(sections) on are copied).  Pair i
    turns by positions[axis of i] * theta ** (-2 i / rotary_dim); order
    "blocks" gives axis a the next sections[a] pairs, "round_robin" deals the
    pairs to the axes in turn; pairing "halves" couples channels (i, i +
    rotary_dim / 2), "adjacent" (2 i, 2 i + 1).  inverse turns back (and is the
    gradient).  Calls on tensors that require a gradient, or carry a tangent of
    torch.autograd.forward_ad, are differentiable (not through torch.func); the
    gradient is computed on the call's stream, in order with what comes before and
    after it.  q_out / k_out may be q / k (in place), and share no other memory with
    them or each other.  Returns (q_out, k_out)."""
    if _differentiated(q, k):
        if q_out is not None or k_out is not None:
            raise ValueError("q_out / k_out cannot be given where a gradient is needed")
        dev = q.get_device()
        _one_device(max(dev, 0), q, k, positions)
        # autograd runs the backward pass on the stream that is current here, and orders
        # the gradients that come and go with it
        with _on(dev, stream):
            got = _RopeAxes.apply(q, k, positions, tuple(sections), theta, order, pairing, inverse)
        return got if k is not None else (got[0], None)
    return _rope(q, k, positions, sections, theta, order, pairing, inverse, q_out, k_out, stream)


def _rope(q, k, positions, sections, theta, order, pairing, inverse, q_out=None, k_out=None,
          stream=None):
    """rope_axes without derivatives."""
    dev = q.get_device()
    _one_device(max(dev, 0), q, k, positions, q_out, k_out)
    sections = tuple(sections)
    plan = _rope_plan(2 * sum(sections), sections, theta, order, pairing)
    with _on(dev, stream) as s:
        qx = _heads("q", q)
        T, Hq, D = qx.shape
        kx = None if k is None else _heads("k", k)
        if kx is not None and (kx.shape[0] != T or kx.shape[2] != D or kx.dtype != qx.dtype):
            raise ValueError("k must have q's tokens, channels and type")
        if (positions.dtype is not torch.int32 or positions.shape != (len(sections), T) or
                (T > 1 and positions.stride(1) != 1)):
            raise ValueError(f"positions must be an int32 [{len(sections)}, {T}] tensor")
        if kx is None and k_out is not None:
            raise ValueError("k_out without k")
        given = q_out, k_out
        if q_out is not None or k_out is not None:
            for o, x in ((q_out, qx), (k_out, kx)):
                if o is not None and (o.shape != x.shape or o.dtype is not x.dtype or
                                      _heads("output", o) is not o):
                    raise ValueError("an output must have its input's shape and type, contiguous "
                                     "channels and strides that are multiples of 8")
            if q_out is not q or k_out is not k or q is k:
                _rope_outputs(qx, kx, q_out, k_out)
        if q_out is None:
            q_out = _like(qx, qx.dtype)
        if kx is not None and k_out is None:
            k_out = _like(kx, kx.dtype)
        qst, qos = qx.stride(), q_out.stride()
        Hk, kst, kos = 0, (0, 0), (0, 0)
        if kx is not None:
            Hk, kst, kos = kx.shape[1], kx.stride(), k_out.stride()
        strides = _I64x8(qst[0], qst[1], kst[0], kst[1], qos[0], qos[1], kos[0], kos[1])
        L.check("tkv_rope_axes", L.lib().tkv_rope_axes(
            C.byref(plan), qx.data_ptr(), None if kx is None else kx.data_ptr(),
            q_out.data_ptr(), None if kx is None else k_out.data_ptr(), _DT[qx.dtype], Hq, Hk, D,
            T, strides, positions.data_ptr(), positions.stride(0), 1 if inverse else 0, s))
    if given != (None, None):
        _written(*given)
    return q_out, k_out


class _RopeAxes(torch.autograd.Function):
    """A rotation is linear: its gradient is the rotation back, a tangent turns as
    the input does.  (rope_axes in both, so they have derivatives of their own.)"""

    @staticmethod
    def forward(ctx, q, k, positions, *how):
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
        *ctx.how, ctx.inverse = how
        ctx.has_k = k is not None
        got = _rope(q, k, positions, *how)
        return got if ctx.has_k else got[:1]

    @staticmethod
    def backward(ctx, *grads):
        (positions,) = ctx.saved_tensors
        gq, gk = rope_axes(grads[0], grads[1] if ctx.has_k else None, positions, *ctx.how,
                           not ctx.inverse)
        return gq, gk, None, None, None, None, None, None

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        (positions,) = ctx.saved_tensors
        turn = lambda t: None if t is None else rope_axes(  # noqa: E731
            t, None, positions, *ctx.how, ctx.inverse)[0]
        return (turn(tq), turn(tk)) if ctx.has_k else (turn(tq),)


class Int8PagedCache:
    """Device buffer of one layer's paged int8 cache: pool [num_pages,
    n_kv_heads, page_bytes] uint8, allocated zeroed, or the caller's (pool=).  A
    page is pool[i]: pool[dst] = pool[src] copies it (a sequence that forks inside
    a page), pool[i].cpu() takes it to the host."""

    def __init__(self, n_kv_heads: int, head_dim: int, num_pages: Optional[int] = None,
                 device="cuda", pool: Optional[torch.Tensor] = None):
        self.n_kv_heads, self.head_dim = int(n_kv_heads), int(head_dim)
        self.page_bytes = int(L.lib().tkv_int8_page_bytes(self.head_dim))
        if not self.page_bytes:
            raise ValueError(f"head_dim {head_dim}: 64 and 128 are supported")
        if (num_pages is None) == (pool is None):
            raise ValueError("give either num_pages or a pool")
        if pool is None:
            pool = torch.zeros((num_pages, self.n_kv_heads, self.page_bytes), dtype=torch.uint8,
                               device=device)
        elif (pool.dtype != torch.uint8 or not pool.is_cuda or not pool.is_contiguous() or
              tuple(pool.shape[1:]) != (self.n_kv_heads, self.page_bytes) or pool.dim() != 3):
            raise ValueError(f"pool must be a contiguous CUDA uint8 [pages, {self.n_kv_heads}, "
                             f"{self.page_bytes}] tensor")
        self.pool = pool
        self.num_pages = int(pool.shape[0])
        self._c = L.TkvInt8Cache(pool.data_ptr(), self.num_pages, self.n_kv_heads, self.head_dim, 0)
        self._ref = C.byref(self._c)
        self._device = pool.get_device()

    def c_struct(self) -> L.TkvInt8Cache:
        return self._c


def int8_append(cache: Int8PagedCache, k_new: torch.Tensor, v_new: torch.Tensor,
                cu_new: torch.Tensor, seq_lens_old: torch.Tensor, block_tables: torch.Tensor,
                max_new_tokens: Optional[int] = None, err: Optional[torch.Tensor] = None,
                stream=None) -> None:
    """Quantises K/V as they are written into the int8 pages.

    k_new, v_new: [T, n_kv_heads, D], both fp16 or both bf16, any token and head
    strides that are multiples of 8 (slices of a fused projection are read where
    they lie); cu_new [B+1], seq_lens_old [B], block_tables [B, max_blocks]
    int32; max_new_tokens bounds a sequence's new tokens (default T)."""
    _no_grad_path("int8_append", k_new, v_new)
    dev = cache._device
    _one_device(max(dev, 0), cache.pool, k_new, v_new, cu_new, seq_lens_old, block_tables, err)
    B = _count(seq_lens_old)
    with _on(dev, stream) as s:
        k, v = _heads("k_new", k_new), _heads("v_new", v_new)
        if k.shape != v.shape or k.dtype != v.dtype or k.shape[1:] != (cache.n_kv_heads,
                                                                      cache.head_dim):
            raise ValueError(f"k_new and v_new must both be [tokens, {cache.n_kv_heads}, "
                             f"{cache.head_dim}] of one type")
        T = k.shape[0]
        ks, vs = k.stride(), v.stride()
        bt, mb = _table(block_tables, B)
        L.check("tkv_int8_append", L.lib().tkv_int8_append(
            cache._ref, k.data_ptr(), v.data_ptr(), _DT[k.dtype],
            _I64x4(ks[0], ks[1], vs[0], vs[1]), _index("cu_new", cu_new, (B + 1,)),
            _index("seq_lens_old", seq_lens_old, (B,)), bt, mb, B, T,
            T if max_new_tokens is None else _i32("max_new_tokens", max_new_tokens), _err_ptr(err),
            s))


def int8_read(cache: Int8PagedCache, block_tables: torch.Tensor, starts: torch.Tensor,
              cu: torch.Tensor, total_tokens: int, max_tokens: Optional[int] = None,
              dtype: torch.dtype = torch.float16, k_out: Optional[torch.Tensor] = None,
              v_out: Optional[torch.Tensor] = None, err: Optional[torch.Tensor] = None,
              stream=None):
    """Reads tokens back from the int8 pages: row cu[s] + i of the returned K
    and V ([total_tokens, n_kv_heads, D] fp16, bf16 or fp32) is token starts[s]
    + i of sequence s.  Rows outside the sequences are not written."""
    dev = cache._device
    _one_device(max(dev, 0), cache.pool, block_tables, starts, cu, k_out, v_out, err)
    B = _count(starts)
    shape = (_i32("total_tokens", total_tokens), cache.n_kv_heads, cache.head_dim)
    with _on(dev, stream) as s:
        if k_out is not None or v_out is not None:
            dtype = (v_out if k_out is None else k_out).dtype
            for t in (k_out, v_out):
                if t is not None and (t.shape != shape or t.dtype is not dtype or
                                      not t.is_contiguous()):
                    raise ValueError(f"k_out / v_out must be contiguous {list(shape)} tensors "
                                     "of one type")
            _plain("k_out", k_out)
            _plain("v_out", v_out)
            if k_out is not None and v_out is not None and not _apart(k_out, v_out):
                raise ValueError("k_out overlaps v_out")
        if dtype not in _DT:
            raise ValueError("dtype must be fp16, bf16 or fp32")
        given = k_out, v_out
        if k_out is None:
            k_out = torch.empty(shape, dtype=dtype, device=cache.pool.device)
        if v_out is None:
            v_out = _like(k_out, dtype)
        bt, mb = _table(block_tables, B)
        L.check("tkv_int8_read", L.lib().tkv_int8_read(
            cache._ref, k_out.data_ptr(), v_out.data_ptr(), _DT[dtype], bt, mb,
            _index("starts", starts, (B,)), _index("cu", cu, (B + 1,)), B, shape[0],
            shape[0] if max_tokens is None else _i32("max_tokens", max_tokens), _err_ptr(err), s))
    if given != (None, None):
        _written(*given)
    return k_out, v_out


def int8_workspace_bytes(num_seqs: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                         max_q_tokens: int, max_context_len: int) -> int:
    sizes = (num_seqs, num_q_heads, num_kv_heads, head_dim, max_q_tokens, max_context_len)
    return int(L.lib().tkv_int8_attend_workspace_bytes(*[_i32("a size", n) for n in sizes]))


def int8_workspace(num_seqs: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                   max_q_tokens: int, max_context_len: int, device="cuda") -> torch.Tensor:
    """Zeroed workspace of int8_attend calls of up to these sizes, on a cache of as
    many kv heads and channels (calls that may overlap on the GPU need one each)."""
    n = int8_workspace_bytes(num_seqs, num_q_heads, num_kv_heads, head_dim, max_q_tokens,
                             max_context_len)
    if n <= 0:
        raise ValueError("sizes out of range")
    return torch.zeros(n, dtype=torch.uint8, device=device)


def int8_attend(cache: Int8PagedCache, q: torch.Tensor, cu_q: torch.Tensor,
                block_tables: torch.Tensor, seq_lens: torch.Tensor,
                max_q_tokens: Optional[int] = None, max_context_len: Optional[int] = None,
                scale: Optional[float] = None, window: int = 0,
                out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                workspace: Optional[torch.Tensor] = None, err: Optional[torch.Tensor] = None,
                stream=None) -> torch.Tensor:
    """Attention of each sequence's last tokens over the int8 pages: rows
    cu_q[s] .. cu_q[s+1] of q [T, Hq, D] (fp16 or bf16, any token and head
    strides that are multiples of 8) are the last tokens of sequence s, already
    appended; each attends to itself and the tokens before it, or to the last
    `window` of them.  One row a sequence is a decode step.  Returns out [T, Hq,
    D] (fp16 or bf16; it may be q, contiguous, and shares no other memory with it); its
    rows outside the sequences are not written."""
    _no_grad_path("int8_attend", q)
    dev = cache._device
    _one_device(max(dev, 0), cache.pool, q, cu_q, block_tables, seq_lens, out, workspace, err)
    B = _count(seq_lens)
    with _on(dev, stream) as s:
        x = _heads("q", q)
        T, Hq, D = x.shape
        if D != cache.head_dim:
            raise ValueError(f"q has {D} channels, the cache {cache.head_dim}")
        if Hq % cache.n_kv_heads:
            raise ValueError(f"{Hq} q heads do not share {cache.n_kv_heads} kv heads evenly")
        bt, mb = _table(block_tables, B)
        mq = T if max_q_tokens is None else _i32("max_q_tokens", max_q_tokens)
        ml = _i32("max_context_len",
                  mb * L.TKV_PAGE_SIZE if max_context_len is None else max_context_len)
        given = out
        if out is None:
            out = _like(x, out_dtype or x.dtype)
        elif out.shape != (T, Hq, D) or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {[T, Hq, D]} tensor")
        if out.dtype not in _HALF:
            raise ValueError("out must be fp16 or bf16")
        if given is not None:
            _plain("out", out)
            if not (_apart(out, x) or _same(out, x)):
                raise ValueError("out overlaps q")
        if workspace is None:
            workspace = int8_workspace(B, Hq, cache.n_kv_heads, D, mq, ml, x.device)
        elif not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")
        st = x.stride()
        L.check("tkv_int8_attend", L.lib().tkv_int8_attend(
            cache._ref, x.data_ptr(), _DT[x.dtype], _I64x2(st[0], st[1]),
            out.data_ptr(), _DT[out.dtype], _index("cu_q", cu_q, (B + 1,)), bt, mb,
            _index("seq_lens", seq_lens, (B,)), B, Hq, T, mq, ml, _i32("window", window),
            1.0 / math.sqrt(D) if scale is None else float(scale), workspace.data_ptr(),
            workspace.nbytes, _err_ptr(err), s))
    if given is not None:
        _written(given)
    return out
