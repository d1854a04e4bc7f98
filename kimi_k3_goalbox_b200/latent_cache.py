"""Operators on the paged latent cache of one MLA layer (include/kk3.h, kk3_cache_*).

What a serving program needs around the decode step: `append` writes the new tokens' entries, `attend` attends any
number of new tokens per sequence, `attention_mass` accumulates the weight that each cached position gets, `evict`
cuts sequences down to the positions that carry it. A step cache [B, capacity, 512] is a paged cache: see
`paged_view`; what these operators leave in it is what `StepContext.step_append` continues.

A cache is three tensors: `kv` bf16 [pages, page_size, 512], `pe` bf16 [pages, page_size, 64] and `table` int32
[B, columns]; position p of sequence b is slot p % page_size of page table[b, p // page_size]. `cu_new` int32 [B + 1]
gives the packed rows of each sequence's new tokens, `lengths` int64 [B] the cached positions (as the step's
`cache_length`). All on one CUDA device; calls are enqueued on that device's current stream, allocate only through
torch's allocator, never synchronise and can be captured into a graph. Device-side values are not read by the host: a
page number outside the pool or a length outside the table reads as zeros, is not written, and sets `error_word`
(optional int32 tensor, zeroed by the caller) to a nonzero code. There is no CPU path: without the library or a GPU
these raise.
"""

from __future__ import annotations

import ctypes

import torch

from .runtime import KK3Error, load_library

LATENT, ROPE = 512, 64
DEFAULT_SCALE = (128 + 64) ** -0.5      # (qk_nope_dim + qk_rope_dim) ** -0.5 (megabench/tasks/kimi.py:278)
MAX_SEQUENCES, MAX_HEADS, MAX_PAGE, MAX_POSITIONS = 4096, 128, 65536, 1 << 27


class CacheDesc(ctypes.Structure):
    """kk3_cache (include/kk3.h)."""
    _fields_ = [("kv", ctypes.c_void_p), ("pe", ctypes.c_void_p), ("kv_page_stride", ctypes.c_int64),
                ("kv_row_stride", ctypes.c_int64), ("pe_page_stride", ctypes.c_int64),
                ("pe_row_stride", ctypes.c_int64), ("table", ctypes.c_void_p), ("table_stride", ctypes.c_int64),
                ("num_pages", ctypes.c_int32), ("page_size", ctypes.c_int32), ("columns", ctypes.c_int32),
                ("batch", ctypes.c_int32)]


_LIB = None


def _lib() -> ctypes.CDLL:
    global _LIB
    if _LIB is None:
        lib = load_library()
        vp, i32, i64, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
        desc = ctypes.POINTER(CacheDesc)
        lib.kk3_cache_append.argtypes = [desc, vp, i64, vp, f32, vp, vp, i32, vp, vp, vp]
        lib.kk3_cache_attend_workspace.argtypes = [i32, i32, i32]
        lib.kk3_cache_attend_workspace.restype = i64
        lib.kk3_cache_attend.argtypes = [desc, vp, i64, i64, vp, i64, i64, vp, vp, i32, i32, f32, vp, vp, vp, i64, vp, vp]
        lib.kk3_cache_mass_workspace.argtypes = [i32, i32, i32]
        lib.kk3_cache_mass_workspace.restype = i64
        lib.kk3_cache_mass.argtypes = [desc, vp, i64, i64, vp, i64, i64, vp, vp, vp, i32, i32, f32, vp, i64, vp, vp, i64,
                                       vp, vp]
        lib.kk3_cache_evict.argtypes = [desc, vp, vp, i64, i32, i32, i32, vp, i64, i32, vp, vp, vp, vp, vp]
        _LIB = lib
    return _LIB


def paged_view(kv_cache: torch.Tensor, pe_cache: torch.Tensor, page_size: int):
    """The step's contiguous caches [B, capacity, 512] / [B, capacity, 64] as a paged cache without a copy:
    (kv, pe, table). capacity must be a multiple of page_size."""
    B, capacity = kv_cache.shape[:2]
    if page_size < 1 or capacity % page_size or pe_cache.shape[:2] != kv_cache.shape[:2]:
        raise ValueError("the capacity must be a multiple of page_size, and the caches must agree")
    columns = capacity // page_size
    table = torch.arange(B * columns, dtype=torch.int32, device=kv_cache.device).view(B, columns)
    return kv_cache.view(-1, page_size, kv_cache.shape[2]), pe_cache.view(-1, page_size, pe_cache.shape[2]), table


# --- argument checks -------------------------------------------------------------------------------------------

def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _on(t, name: str, device: torch.device, dtype: torch.dtype, shape: tuple) -> torch.Tensor:
    _need(isinstance(t, torch.Tensor), f"{name} must be a tensor")
    _need(t.device == device, f"{name} must be on {device}, with the cache")
    _need(t.dtype == dtype and tuple(t.shape) == shape, f"{name} must be {dtype} {list(shape)}")
    return t


def _rows16(t: torch.Tensor, name: str) -> None:
    """Vector loads: last dim contiguous, the other strides multiples of 8 elements, 16-byte aligned."""
    _need(t.stride(-1) == 1 and all(s % 8 == 0 and s >= 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1)
          and t.data_ptr() % 16 == 0,
          f"{name} needs a contiguous last dim, strides that are multiples of 8 elements and 16-byte alignment")


def _stride(t: torch.Tensor, dim: int) -> int:
    """A stride for the kernels; that of a dim of one element means nothing and is made a valid one."""
    return t.stride(dim) if t.shape[dim] > 1 else (t.shape[-1] + 7) // 8 * 8


def _cache(kv, pe, table) -> tuple[CacheDesc, torch.device, int]:
    """(descriptor, device, positions per sequence)."""
    for t, name in ((kv, "kv"), (pe, "pe"), (table, "table")):
        _need(isinstance(t, torch.Tensor), f"{name} must be a tensor")
    _need(kv.is_cuda, "the cache must be on a CUDA device (sm_100a kernels, no CPU path)")
    _need(kv.dim() == 3 and kv.dtype == torch.bfloat16 and kv.shape[2] == LATENT and kv.shape[0] > 0 and kv.shape[1] > 0,
          "kv must be bfloat16 [pages, page_size, 512]")
    _on(pe, "pe", kv.device, torch.bfloat16, (kv.shape[0], kv.shape[1], ROPE))
    _need(table.dim() == 2 and min(table.shape) > 0, "table must be int32 [B, columns], not empty")
    _on(table, "table", kv.device, torch.int32, tuple(table.shape))
    _need(table.stride(1) == 1 or table.shape[1] == 1, "table rows must be contiguous")
    _rows16(kv, "kv")
    _rows16(pe, "pe")
    pages, page = kv.shape[:2]
    B, columns = table.shape
    _need(B <= MAX_SEQUENCES and page <= MAX_PAGE and columns * page <= MAX_POSITIONS and pages < 1 << 31,
          f"at most {MAX_SEQUENCES} sequences, pages of {MAX_PAGE} and {MAX_POSITIONS} positions per sequence")
    for t, name in ((kv, "kv"), (pe, "pe")):
        _need(t.shape[1] == 1 or t.stride(1) >= t.shape[2], f"{name} rows must not overlap")
    desc = CacheDesc(kv.data_ptr(), pe.data_ptr(), _stride(kv, 0), _stride(kv, 1), _stride(pe, 0), _stride(pe, 1),
                     table.data_ptr(), table.stride(0) if B > 1 else columns, pages, page, columns, B)
    return desc, kv.device, columns * page


def _error(error_word, device) -> int | None:
    if error_word is None:
        return None
    _need(isinstance(error_word, torch.Tensor) and error_word.device == device and error_word.dtype == torch.int32
          and error_word.numel() == 1, "error_word must be one int32 on the cache's device")
    return error_word.data_ptr()


def _queries(q_latent, q_pe, device, scale):
    _need(isinstance(q_latent, torch.Tensor) and q_latent.dim() == 3, "q_latent must be bfloat16 [T, heads, 512]")
    T, H = q_latent.shape[:2]
    _need(1 <= H <= MAX_HEADS, f"heads must be 1..{MAX_HEADS}")
    _need(T * H < 1 << 30, "too many query rows")
    _on(q_latent, "q_latent", device, torch.bfloat16, (T, H, LATENT))
    _on(q_pe, "q_pe", device, torch.bfloat16, (T, H, ROPE))
    if T:
        _rows16(q_latent, "q_latent")
        _rows16(q_pe, "q_pe")
    scale = DEFAULT_SCALE if scale is None else float(scale)
    _need(scale == scale and abs(scale) != float("inf"), "scale must be finite")
    args = (q_latent.data_ptr(), _stride(q_latent, 0), _stride(q_latent, 1), q_pe.data_ptr(), _stride(q_pe, 0),
            _stride(q_pe, 1))
    return T, H, scale, args


def _call(rc: int, what: str) -> None:
    if rc != 0:
        raise KK3Error(rc, what)


def _stream(device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


# --- the operators ---------------------------------------------------------------------------------------------

def append(raw, norm_weight, kv, pe, table, lengths, cu_new, *, eps: float = 1e-6, error_word=None) -> torch.Tensor:
    """Write the new tokens' entries behind their sequences and return the new lengths (int64 [B]).

    raw: bf16 [T, 576], the `ka` projection of the new tokens; its first 512 values are RMS-normalised with
    norm_weight (bf16 [512]) in FP32 and rounded once, the other 64 are stored as they are. lengths: positions cached
    before. A token behind the table's last column is not written and sets error_word."""
    desc, dev, _ = _cache(kv, pe, table)
    _need(isinstance(raw, torch.Tensor) and raw.dim() == 2, "raw must be bfloat16 [T, 576]")
    T = raw.shape[0]
    _on(raw, "raw", dev, torch.bfloat16, (T, LATENT + ROPE))
    if T:
        _rows16(raw, "raw")
    _on(norm_weight, "norm_weight", dev, torch.bfloat16, (LATENT,))
    _rows16(norm_weight, "norm_weight")
    _on(lengths, "lengths", dev, torch.int64, (desc.batch,))
    _on(cu_new, "cu_new", dev, torch.int32, (desc.batch + 1,))
    _need(lengths.is_contiguous() and cu_new.is_contiguous(), "lengths and cu_new must be contiguous")
    _need(eps >= 0, "eps must not be negative")
    err = _error(error_word, dev)
    with torch.cuda.device(dev):
        out = torch.empty_like(lengths)
        _call(_lib().kk3_cache_append(ctypes.byref(desc), raw.data_ptr(), _stride(raw, 0), norm_weight.data_ptr(), eps,
                                      lengths.data_ptr(), cu_new.data_ptr(), T, out.data_ptr(), err, _stream(dev)),
              "kk3_cache_append")
    return out


def attend(q_latent, q_pe, kv, pe, table, lengths, cu_new, *, scale: float | None = None, out=None, lse=None,
           error_word=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of the new tokens over their sequences' caches, in the latent space: (out bf16 [T, heads, 512],
    lse f32 [T, heads]).

    q_latent: bf16 [T, heads, 512] absorbed queries, q_pe: bf16 [T, heads, 64]; any strides that are multiples of 8.
    lengths: cached positions, the new tokens included (append's result): token i of n sees the first
    lengths - n + i + 1. A token that sees nothing gets zeros and -inf. Rows behind cu_new[B] are not written (pass
    `out` and `lse`, both contiguous, to keep theirs)."""
    desc, dev, _ = _cache(kv, pe, table)
    T, H, scale, q = _queries(q_latent, q_pe, dev, scale)
    _on(lengths, "lengths", dev, torch.int64, (desc.batch,))
    _on(cu_new, "cu_new", dev, torch.int32, (desc.batch + 1,))
    _need(lengths.is_contiguous() and cu_new.is_contiguous(), "lengths and cu_new must be contiguous")
    err = _error(error_word, dev)
    with torch.cuda.device(dev):
        if out is None:
            out = torch.empty((T, H, LATENT), dtype=torch.bfloat16, device=dev)
        if lse is None:
            lse = torch.empty((T, H), dtype=torch.float32, device=dev)
        _on(out, "out", dev, torch.bfloat16, (T, H, LATENT))
        _on(lse, "lse", dev, torch.float32, (T, H))
        _need(out.is_contiguous() and lse.is_contiguous() and out.data_ptr() % 16 == 0,
              "out and lse must be contiguous, out 16-byte aligned")
        if T == 0:
            return out, lse
        lib = _lib()
        nbytes = lib.kk3_cache_attend_workspace(desc.batch, T, H)
        work = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=dev)
        _call(lib.kk3_cache_attend(ctypes.byref(desc), *q, lengths.data_ptr(), cu_new.data_ptr(), T, H, scale,
                                   out.data_ptr(), lse.data_ptr(), work.data_ptr(), nbytes, err, _stream(dev)),
              "kk3_cache_attend")
    return out, lse


def attention_mass(q_latent, q_pe, lse, kv, pe, table, lengths, cu_new, *, scale: float | None = None, mass=None,
                   out=None, error_word=None) -> torch.Tensor:
    """The attention weight that each cached position gets from the new tokens, summed over tokens and heads and added
    to `mass`: f32 [B, columns * page_size].

    lse: attend's, with the same queries, lengths and scale. mass: what earlier calls accumulated (zeros if None);
    `out` may be mass itself. Positions at or behind a length keep their mass."""
    desc, dev, capacity = _cache(kv, pe, table)
    T, H, scale, q = _queries(q_latent, q_pe, dev, scale)
    _on(lse, "lse", dev, torch.float32, (T, H))
    _on(lengths, "lengths", dev, torch.int64, (desc.batch,))
    _on(cu_new, "cu_new", dev, torch.int32, (desc.batch + 1,))
    _need(lengths.is_contiguous() and cu_new.is_contiguous() and lse.is_contiguous(),
          "lengths, cu_new and lse must be contiguous")
    if mass is not None:
        _on(mass, "mass", dev, torch.float32, (desc.batch, capacity))
        _need(mass.stride(1) == 1 or capacity == 1, "mass rows must be contiguous")
    err = _error(error_word, dev)
    with torch.cuda.device(dev):
        if out is None:
            out = torch.empty((desc.batch, capacity), dtype=torch.float32, device=dev)
        _on(out, "out", dev, torch.float32, (desc.batch, capacity))
        _need(out.is_contiguous(), "out must be contiguous")
        lib = _lib()
        nbytes = lib.kk3_cache_mass_workspace(desc.batch, T, H)
        work = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=dev)
        _call(lib.kk3_cache_mass(ctypes.byref(desc), *q, lse.data_ptr(), lengths.data_ptr(), cu_new.data_ptr(), T, H,
                                 scale, None if mass is None else mass.data_ptr(),
                                 0 if mass is None else (mass.stride(0) if desc.batch > 1 else capacity),
                                 out.data_ptr(), work.data_ptr(), nbytes, err, _stream(dev)), "kk3_cache_mass")
    return out


def evict(kv, pe, table, lengths, mass, budget: int, *, sinks: int = 0, recent: int = 0, dst_table=None,
          error_word=None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cut every sequence down to `budget` positions: its first `sinks`, its last `recent`, and of the others those of
    the largest mass (equal ones: the lowest position; NaN counts as the largest).

    The kept entries move, in ascending order, to positions 0, 1, ... of dst_table's pages (int32 [B, columns2]; pages
    that none of the sequences uses, so that pages shared with others stay as they are), or in place (None). Returns
    (new lengths int64 [B], their mass f32 [B, columns * page_size] with zeros behind, their old positions int32
    [B, budget] with -1 behind)."""
    desc, dev, capacity = _cache(kv, pe, table)
    _on(lengths, "lengths", dev, torch.int64, (desc.batch,))
    _need(lengths.is_contiguous(), "lengths must be contiguous")
    _on(mass, "mass", dev, torch.float32, (desc.batch, capacity))
    _need(mass.stride(1) == 1 or capacity == 1, "mass rows must be contiguous")
    budget, sinks, recent = int(budget), int(sinks), int(recent)
    _need(1 <= budget <= capacity, "budget must be 1 .. columns * page_size")
    _need(sinks >= 0 and recent >= 0 and sinks + recent <= budget, "sinks + recent must not exceed the budget")
    dst, dst_stride, dst_columns = None, 0, 0
    if dst_table is not None:
        _need(isinstance(dst_table, torch.Tensor) and dst_table.dim() == 2, "dst_table must be int32 [B, columns]")
        dst_columns = dst_table.shape[1]
        _on(dst_table, "dst_table", dev, torch.int32, (desc.batch, dst_columns))
        _need(dst_table.stride(1) == 1 or dst_columns == 1, "dst_table rows must be contiguous")
        _need(min(dst_columns * desc.page_size, MAX_POSITIONS) >= budget, "dst_table must hold the budget")
        dst, dst_stride = dst_table.data_ptr(), dst_table.stride(0) if desc.batch > 1 else dst_columns
    err = _error(error_word, dev)
    with torch.cuda.device(dev):
        new_lengths = torch.empty_like(lengths)
        new_mass = torch.empty((desc.batch, capacity), dtype=torch.float32, device=dev)
        kept = torch.empty((desc.batch, budget), dtype=torch.int32, device=dev)
        _call(_lib().kk3_cache_evict(ctypes.byref(desc), lengths.data_ptr(), mass.data_ptr(),
                                     mass.stride(0) if desc.batch > 1 else capacity, budget, sinks, recent, dst,
                                     dst_stride, dst_columns, new_lengths.data_ptr(), new_mass.data_ptr(),
                                     kept.data_ptr(), err, _stream(dev)), "kk3_cache_evict")
    return new_lengths, new_mass, kept
