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
import struct

import torch

from .runtime import KK3Error, load_library

LATENT, ROPE = 512, 64
DEFAULT_SCALE = (128 + 64) ** -0.5      # (qk_nope_dim + qk_rope_dim) ** -0.5 (megabench/tasks/kimi.py:278)
MAX_SEQUENCES, MAX_HEADS, MAX_PAGE, MAX_POSITIONS = 4096, 128, 65536, 1 << 27


# kk3_cache (include/kk3.h) as bytes: kv, pe, their page and row strides, table, table_stride, num_pages, page_size,
# columns, batch
_DESC = struct.Struct("=QQqqqqQqiiii")


_LIB = None
_raw_stream = torch._C._cuda_getCurrentRawStream    # current_stream(device).cuda_stream without the Stream object


def _lib() -> ctypes.CDLL:
    global _LIB
    if _LIB is None:
        lib = load_library()
        vp, i32, i64, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
        desc = ctypes.c_char_p
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
# A decode step calls these operators once per layer, so the checks are written to cost little when they pass: one
# comparison a line, and a message is only put together for a refusal.

_BF16, _F32, _I32, _I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _check(t, name: str, device: torch.device, dtype: torch.dtype, shape: tuple) -> None:
    """`t` is a contiguous tensor of this kind."""
    _check_kind(t, name, device, dtype, shape)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _check_kind(t, name: str, device: torch.device, dtype: torch.dtype, shape: tuple) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if t.dtype != dtype or t.shape != shape:
        raise ValueError(f"{name} must be {dtype} {list(shape)}, not {t.dtype} {list(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, with the cache")


def _vector_rows(t, name: str) -> None:
    """Refuse what 16-byte loads cannot read."""
    if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s % 8 or s < 0 for n, s in zip(t.shape[:-1], t.stride()) if n > 1):
        raise ValueError(f"{name} needs a contiguous last dim, strides that are multiples of 8 elements and 16-byte "
                         "alignment")


def _strides3(t, name: str) -> tuple[int, int, int]:
    """(address, strides of the first two dims) of a three-dimensional tensor that the kernels read with 16-byte loads.
    The stride of a dim of one element means nothing and is made a valid one."""
    s0, s1, s2 = t.stride()
    n0, n1, n2 = t.shape
    at = t.data_ptr()
    if s2 != 1 or (at | s0 * 2 | s1 * 2) & 15 or s0 < 0 or s1 < 0:
        _vector_rows(t, name)
    return at, s0 if n0 > 1 else n1 * n2, s1 if n1 > 1 else n2


def _query_rows(t):
    """(tensor, token stride, head stride) of queries [T, heads, n] whose (token, head) rows lie at one pitch, 16-byte
    aligned, as the kernels' copies need; others are copied into that form."""
    s0, s1, s2 = t.stride()
    n0, n1, n2 = t.shape
    if n1 == 1:
        s1 = n2 if n0 == 1 else s0
    if s2 != 1 or s1 < n2 or s1 % 8 or (n0 > 1 and s0 != n1 * s1) or t.data_ptr() % 16:
        return t.clone(memory_format=torch.contiguous_format), n1 * n2, n2
    return t, n1 * s1, s1


def _cache(kv, pe, table):
    """(kk3_cache bytes, device, sequences, positions per sequence)."""
    if not isinstance(kv, torch.Tensor) or kv.dim() != 3 or kv.dtype != _BF16 or kv.shape[2] != LATENT or 0 in kv.shape:
        raise ValueError("kv must be bfloat16 [pages, page_size, 512], not empty")
    dev = kv.device
    if dev.type != "cuda":
        raise ValueError("the cache must be on a CUDA device (sm_100a kernels, no CPU path)")
    pages, page, _ = kv.shape
    _check_kind(pe, "pe", dev, _BF16, (pages, page, ROPE))
    if not isinstance(table, torch.Tensor) or table.dim() != 2 or 0 in table.shape:
        raise ValueError("table must be int32 [B, columns], not empty")
    B, columns = table.shape
    _check_kind(table, "table", dev, _I32, (B, columns))
    kv_at, kv_page, kv_row = _strides3(kv, "kv")
    pe_at, pe_page, pe_row = _strides3(pe, "pe")
    if kv_row < LATENT or pe_row < ROPE:
        raise ValueError("the rows of kv and pe must not overlap")
    if page > 1 and (kv_page % kv_row or pe_page % pe_row):
        raise ValueError("the page strides of kv and pe must be multiples of their row strides")
    if columns > 1 and table.stride(1) != 1:
        raise ValueError("table rows must be contiguous")
    if B > MAX_SEQUENCES or page > MAX_PAGE or columns * page > MAX_POSITIONS or pages >= 1 << 31:
        raise ValueError(f"at most {MAX_SEQUENCES} sequences, pages of {MAX_PAGE} and {MAX_POSITIONS} positions per "
                         "sequence")
    desc = _DESC.pack(kv_at, pe_at, kv_page, kv_row, pe_page, pe_row, table.data_ptr(),
                      table.stride(0) if B > 1 else columns, pages, page, columns, B)
    return desc, dev, B, columns * page


def _error(error_word, device) -> int | None:
    if error_word is None:
        return None
    _need(isinstance(error_word, torch.Tensor) and error_word.device == device and error_word.dtype == _I32
          and error_word.numel() == 1, "error_word must be one int32 on the cache's device")
    return error_word.data_ptr()


def _queries(q_latent, q_pe, device, scale):
    if not isinstance(q_latent, torch.Tensor) or q_latent.dim() != 3:
        raise ValueError("q_latent must be bfloat16 [T, heads, 512]")
    T, H, _ = q_latent.shape
    if not 1 <= H <= MAX_HEADS or T * H >= 1 << 30:
        raise ValueError(f"heads must be 1..{MAX_HEADS}, and T * heads below 2^30")
    _check_kind(q_latent, "q_latent", device, _BF16, (T, H, LATENT))
    _check_kind(q_pe, "q_pe", device, _BF16, (T, H, ROPE))
    scale = DEFAULT_SCALE if scale is None else float(scale)
    if scale != scale or abs(scale) == float("inf"):
        raise ValueError("scale must be finite")
    if T:
        q_latent, *ql = _query_rows(q_latent)
        q_pe, *qp = _query_rows(q_pe)
    else:
        ql, qp = (LATENT, LATENT), (ROPE, ROPE)
    return T, H, scale, (q_latent, q_pe), (q_latent.data_ptr(), *ql, q_pe.data_ptr(), *qp)


def _mass_stride(mass, name: str, device, B: int, capacity: int) -> int:
    _check_kind(mass, name, device, _F32, (B, capacity))
    row, one = mass.stride()
    if (one != 1 and capacity > 1) or row < 0:
        raise ValueError(f"{name} rows must be contiguous")
    return row if B > 1 else capacity


def _run(what: str, device: torch.device, *args) -> None:
    """Call a C entry point on the cache's device and its current stream."""
    fn, index = getattr(_lib(), what), device.index
    if torch.cuda.current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc != 0:
        raise KK3Error(rc, what)


def _workspace(what: str, device: torch.device, *args) -> torch.Tensor:
    """A call's own workspace, from torch's allocator on the current stream."""
    if torch.cuda.current_device() == device.index:
        nbytes = getattr(_lib(), what)(*args)
    else:
        with torch.cuda.device(device):
            nbytes = getattr(_lib(), what)(*args)
    if nbytes <= 0:
        raise KK3Error(-3, what)
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


# --- the operators ---------------------------------------------------------------------------------------------

def append(raw, norm_weight, kv, pe, table, lengths, cu_new, *, eps: float = 1e-6, error_word=None) -> torch.Tensor:
    """Write the new tokens' entries behind their sequences and return the new lengths (int64 [B]).

    raw: bf16 [T, 576], the `ka` projection of the new tokens; its first 512 values are RMS-normalised with
    norm_weight (bf16 [512]) in FP32 and rounded once, the other 64 are stored as they are. lengths: positions cached
    before. A token behind the table's last column is not written and sets error_word."""
    desc, dev, B, _ = _cache(kv, pe, table)
    if not isinstance(raw, torch.Tensor) or raw.dim() != 2:
        raise ValueError("raw must be bfloat16 [T, 576]")
    T = raw.shape[0]
    _check_kind(raw, "raw", dev, _BF16, (T, LATENT + ROPE))
    _check(norm_weight, "norm_weight", dev, _BF16, (LATENT,))
    _vector_rows(norm_weight, "norm_weight")
    _check(lengths, "lengths", dev, _I64, (B,))
    _check(cu_new, "cu_new", dev, _I32, (B + 1,))
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    row = LATENT + ROPE
    if T:
        _vector_rows(raw, "raw")
        row = raw.stride(0) if T > 1 else row
    out = torch.empty_like(lengths)
    _run("kk3_cache_append", dev, desc, raw.data_ptr(), row, norm_weight.data_ptr(), eps, lengths.data_ptr(),
         cu_new.data_ptr(), T, out.data_ptr(), _error(error_word, dev))
    return out


def attend(q_latent, q_pe, kv, pe, table, lengths, cu_new, *, scale: float | None = None, out=None, lse=None,
           error_word=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of the new tokens over their sequences' caches, in the latent space: (out bf16 [T, heads, 512],
    lse f32 [T, heads]).

    q_latent: bf16 [T, heads, 512] absorbed queries, q_pe: bf16 [T, heads, 64], of any strides (unless
    all (token, head) rows lie at one 16-byte aligned pitch, they are copied first).
    lengths: cached positions, the new tokens included (append's result): token i of n sees the first
    lengths - n + i + 1. A token that sees nothing gets zeros and -inf. Rows behind cu_new[B] are not written (pass
    `out` and `lse`, both contiguous, to keep theirs)."""
    desc, dev, B, _ = _cache(kv, pe, table)
    T, H, scale, _copies, q = _queries(q_latent, q_pe, dev, scale)
    _check(lengths, "lengths", dev, _I64, (B,))
    _check(cu_new, "cu_new", dev, _I32, (B + 1,))
    if out is None:
        out = torch.empty((T, H, LATENT), dtype=_BF16, device=dev)
    else:
        _check(out, "out", dev, _BF16, (T, H, LATENT))
        _need(out.data_ptr() % 16 == 0, "out must be 16-byte aligned")
    if lse is None:
        lse = torch.empty((T, H), dtype=_F32, device=dev)
    else:
        _check(lse, "lse", dev, _F32, (T, H))
    err = _error(error_word, dev)
    if T:
        work = _workspace("kk3_cache_attend_workspace", dev, B, T, H)
        _run("kk3_cache_attend", dev, desc, *q, lengths.data_ptr(), cu_new.data_ptr(), T, H, scale, out.data_ptr(),
             lse.data_ptr(), work.data_ptr(), work.numel(), err)
    return out, lse


def attention_mass(q_latent, q_pe, lse, kv, pe, table, lengths, cu_new, *, scale: float | None = None, mass=None,
                   out=None, error_word=None) -> torch.Tensor:
    """The attention weight that each cached position gets from the new tokens, summed over tokens and heads and added
    to `mass`: f32 [B, columns * page_size].

    lse: attend's, with the same queries, lengths and scale. mass: what earlier calls accumulated (zeros if None);
    `out` may be mass itself. Positions at or behind a length keep their mass."""
    desc, dev, B, capacity = _cache(kv, pe, table)
    T, H, scale, _copies, q = _queries(q_latent, q_pe, dev, scale)
    _check(lse, "lse", dev, _F32, (T, H))
    _check(lengths, "lengths", dev, _I64, (B,))
    _check(cu_new, "cu_new", dev, _I32, (B + 1,))
    row, before = 0, None
    if mass is not None:
        row, before = _mass_stride(mass, "mass", dev, B, capacity), mass.data_ptr()
    if out is None:
        out = torch.empty((B, capacity), dtype=_F32, device=dev)
    else:
        _check(out, "out", dev, _F32, (B, capacity))
    work = _workspace("kk3_cache_mass_workspace", dev, B, T, H)
    _run("kk3_cache_mass", dev, desc, *q, lse.data_ptr(), lengths.data_ptr(), cu_new.data_ptr(), T, H, scale, before, row,
         out.data_ptr(), work.data_ptr(), work.numel(), _error(error_word, dev))
    return out


def evict(kv, pe, table, lengths, mass, budget: int, *, sinks: int = 0, recent: int = 0, dst_table=None,
          error_word=None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cut every sequence down to `budget` positions: its first `sinks`, its last `recent`, and of the others those of
    the largest mass (equal ones: the lowest position; NaN counts as the largest).

    The kept entries move, in ascending order, to positions 0, 1, ... of dst_table's pages (int32 [B, columns2]; pages
    that none of the sequences uses, so that pages shared with others stay as they are), or in place (None). Returns
    (new lengths int64 [B], their mass f32 [B, columns * page_size] with zeros behind, their old positions int32
    [B, budget] with -1 behind)."""
    desc, dev, B, capacity = _cache(kv, pe, table)
    _check(lengths, "lengths", dev, _I64, (B,))
    row = _mass_stride(mass, "mass", dev, B, capacity)
    budget, sinks, recent = int(budget), int(sinks), int(recent)
    if not 1 <= budget <= capacity:
        raise ValueError("budget must be 1 .. columns * page_size")
    if sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError("sinks + recent must not exceed the budget")
    dst, dst_row, dst_columns = None, 0, 0
    if dst_table is not None:
        if not isinstance(dst_table, torch.Tensor) or dst_table.dim() != 2:
            raise ValueError("dst_table must be int32 [B, columns]")
        dst_columns = dst_table.shape[1]
        _check_kind(dst_table, "dst_table", dev, _I32, (B, dst_columns))
        if dst_columns > 1 and dst_table.stride(1) != 1:
            raise ValueError("dst_table rows must be contiguous")
        if dst_columns * kv.shape[1] < budget:
            raise ValueError("dst_table must hold the budget")
        dst, dst_row = dst_table.data_ptr(), dst_table.stride(0) if B > 1 else dst_columns
    new_lengths = torch.empty_like(lengths)
    new_mass = torch.empty((B, capacity), dtype=_F32, device=dev)
    kept = torch.empty((B, budget), dtype=_I32, device=dev)
    _run("kk3_cache_evict", dev, desc, lengths.data_ptr(), mass.data_ptr(), row, budget, sinks, recent, dst, dst_row,
         dst_columns, new_lengths.data_ptr(), new_mass.data_ptr(), kept.data_ptr(), _error(error_word, dev))
    return new_lengths, new_mass, kept
