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
(optional int32 tensor, zeroed by the caller) to a nonzero code. Without an error_word such a call is silent, so a
program that fills its tables on the device should pass one and look at it now and then. A wait inside `attend` or
`attention_mass` that runs out (two seconds; a defect, no healthy call comes near it) sets it as well, and the results
that it was for are NaN. Nothing here is differentiable: results carry no gradient, whatever the inputs ask for.
There is no CPU path: without the library or a GPU
these raise.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from .runtime import KK3Error, load_library

LATENT, ROPE = 512, 64
DEFAULT_SCALE = (128 + 64) ** -0.5      # (qk_nope_dim + qk_rope_dim) ** -0.5 (megabench/tasks/kimi.py:278)
MAX_SCALE = 2.35e38                     # its product with log2(e) stays finite in FP32
MAX_SEQUENCES, MAX_HEADS, MAX_PAGE, MAX_POSITIONS = 4096, 128, 65536, 1 << 27


# The argument blocks of include/kk3.h as bytes. kk3_cache: kv, pe, their page and row strides, table, table_stride,
# num_pages, page_size, columns, batch; then each operator's own fields in their order.
_CACHE = "QQqqqqQqiiii"
_APPEND = struct.Struct("=" + _CACHE + "QqQQQQQif")
_ATTEND = struct.Struct("=" + _CACHE + "QqqQqqQQQQQqQiifi")
_MASS = struct.Struct("=" + _CACHE + "QqqQqqQQQQqQQqQiifi")
_EVICT = struct.Struct("=" + _CACHE + "QQqQqQQQQiiii")

_LIB = None
_WORKSPACE: dict = {}       # (operator, device index) -> bytes, the same for every call on a device
_raw_stream = torch._C._cuda_getCurrentRawStream    # current_stream(device).cuda_stream without the Stream object
_current_device = torch.cuda.current_device


def _lib() -> ctypes.CDLL:
    global _LIB
    if _LIB is None:
        lib = load_library()
        for name in ("append", "append_step", "attend", "mass", "evict"):
            getattr(lib, f"kk3_cache_{name}").argtypes = [ctypes.c_char_p, ctypes.c_void_p]
        for name in ("attend", "mass"):
            getattr(lib, f"kk3_cache_{name}_workspace").argtypes = []
            getattr(lib, f"kk3_cache_{name}_workspace").restype = ctypes.c_int64
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
# A decode step calls these operators once per layer, so a check that passes is one expression; what is wrong is only
# looked for, and put into words, when it fails.

_BF16, _F32, _I32, _I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64


def _explain(device, *expected) -> None:
    """Raise for the first of (tensor, name, dtype, shape or None, contiguous) that is not what it should be."""
    for t, name, dtype, shape, contiguous in expected:
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{name} must be a tensor")
        if t.dtype != dtype or (shape is not None and t.shape != shape):
            raise ValueError(f"{name} must be {dtype}{'' if shape is None else ' ' + str(list(shape))}, not {t.dtype} "
                             f"{list(t.shape)}")
    for t, name, _, _, contiguous in expected:
        if not t.is_cuda:
            raise ValueError(f"{name} must be on a CUDA device (sm_100a kernels, no CPU path)")
        if t.get_device() != device:
            raise ValueError(f"{name} must be on cuda:{device}, with the cache")
        if contiguous and not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    raise ValueError("arguments do not fit together")


def _explain_rows(*tensors) -> None:
    for t, name in tensors:
        if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s % 8 or s < 0 for n, s in zip(t.shape[:-1], t.stride()) if n > 1):
            raise ValueError(f"{name} needs a contiguous last dim, strides that are multiples of 8 elements and 16-byte "
                             "alignment")
    raise ValueError("the rows of kv and pe must not overlap, and their page strides must be multiples of their row strides")


def _cache(kv, pe, table):
    """(the fields of kk3_cache, device index, sequences, positions per sequence)."""
    try:
        ks, ts, dev = kv.shape, table.shape, kv.get_device()
        fine = (len(ks) == 3 and len(ts) == 2 and ks[2] == LATENT and kv.dtype is _BF16 and pe.dtype is _BF16
                and table.dtype is _I32 and dev >= 0 and pe.get_device() == dev and table.get_device() == dev
                and pe.shape == (ks[0], ks[1], ROPE) and ks[0] > 0 and ks[1] > 0 and ts[0] > 0 and ts[1] > 0)
    except AttributeError:
        fine = False
    if not fine:
        for t, name, n in ((kv, "kv", 3), (pe, "pe", 3), (table, "table", 2)):
            if not isinstance(t, torch.Tensor) or t.dim() != n or 0 in t.shape:
                raise ValueError(f"{name} must be a tensor of {n} dims, not empty")
        _explain(kv.get_device(), (kv, "kv", _BF16, (kv.shape[0], kv.shape[1], LATENT), False),
                 (pe, "pe", _BF16, (kv.shape[0], kv.shape[1], ROPE), False), (table, "table", _I32, None, False))
    pages, page, _ = ks
    B, columns = ts
    kv_at, pe_at = kv.data_ptr(), pe.data_ptr()
    k0, k1, k2 = kv.stride()
    p0, p1, p2 = pe.stride()
    # the stride of a dim of one element means nothing
    if page == 1:
        k1, p1 = (k0, p0) if pages > 1 else (LATENT, ROPE)
    if pages == 1:
        k0, p0 = page * k1, page * p1
    if (k2 != 1 or p2 != 1 or (kv_at | pe_at) & 15 or (k0 | k1 | p0 | p1) & 7 or k1 < LATENT or p1 < ROPE or k0 < 0 or p0 < 0
            or k0 % k1 or p0 % p1):
        _explain_rows((kv, "kv"), (pe, "pe"))
    t0, t1 = table.stride()
    if (t1 != 1 and columns > 1) or t0 < 0:
        raise ValueError("table rows must be contiguous")
    if B > MAX_SEQUENCES or page > MAX_PAGE or columns * page > MAX_POSITIONS or pages >= 1 << 31:
        raise ValueError(f"at most {MAX_SEQUENCES} sequences, pages of {MAX_PAGE} and {MAX_POSITIONS} positions per "
                         "sequence")
    return (kv_at, pe_at, k0, k1, p0, p1, table.data_ptr(), t0 if B > 1 else columns, pages, page, columns, B), dev, B, columns * page


def _error(error_word, device: int) -> int:
    if error_word is None:
        return 0
    if (not isinstance(error_word, torch.Tensor) or error_word.get_device() != device or error_word.dtype != _I32
            or error_word.numel() != 1):
        raise ValueError("error_word must be one int32 on the cache's device")
    return error_word.data_ptr()


def _query_rows(t):
    """(tensor, token stride, head stride) of queries [T, heads, n] whose (token, head) rows lie at one pitch, 16-byte
    aligned, as the kernels' copies need; others are copied into that form."""
    n0, n1, n2 = t.shape
    if t.is_contiguous() and not t.data_ptr() & 15:
        return t, n1 * n2, n2
    s0, s1, s2 = t.stride()
    if n1 == 1:
        s1 = n2 if n0 == 1 else s0
    if s2 != 1 or s1 < n2 or s1 % 8 or (n0 > 1 and s0 != n1 * s1) or t.data_ptr() % 16:
        return t.clone(memory_format=torch.contiguous_format), n1 * n2, n2
    return t, n1 * s1, s1


def _queries(q_latent, q_pe, lengths, cu_new, dev: int, B: int, scale):
    """(T, heads, scale, tensors to keep until the launch, q_latent and its strides, q_pe and its strides)."""
    try:
        qs = q_latent.shape
        fine = (len(qs) == 3 and qs[2] == LATENT and q_pe.shape == (qs[0], qs[1], ROPE) and q_latent.dtype is _BF16
                and q_pe.dtype is _BF16 and q_latent.get_device() == dev and q_pe.get_device() == dev
                and lengths.dtype is _I64 and cu_new.dtype is _I32 and lengths.shape == (B,) and cu_new.shape == (B + 1,)
                and lengths.get_device() == dev and cu_new.get_device() == dev
                and lengths.is_contiguous() and cu_new.is_contiguous())
    except AttributeError:
        fine = False
    if not fine:
        if not isinstance(q_latent, torch.Tensor) or q_latent.dim() != 3:
            raise ValueError("q_latent must be bfloat16 [T, heads, 512]")
        T, H = q_latent.shape[:2]
        _explain(dev, (q_latent, "q_latent", _BF16, (T, H, LATENT), False), (q_pe, "q_pe", _BF16, (T, H, ROPE), False),
                 (lengths, "lengths", _I64, (B,), True), (cu_new, "cu_new", _I32, (B + 1,), True))
    T, H, _ = qs
    if not 1 <= H <= MAX_HEADS or T * H >= 1 << 30:
        raise ValueError(f"heads must be 1..{MAX_HEADS}, and T * heads below 2^30")
    if scale is None:
        scale = DEFAULT_SCALE
    else:
        scale = float(scale)
        if not abs(scale) <= MAX_SCALE:
            raise ValueError(f"scale must be finite, within {MAX_SCALE}")
    if T:
        q_latent, l0, l1 = _query_rows(q_latent)
        q_pe, p0, p1 = _query_rows(q_pe)
    else:
        l0, l1, p0, p1 = LATENT, LATENT, ROPE, ROPE
    return T, H, scale, (q_latent, q_pe), (q_latent.data_ptr(), l0, l1, q_pe.data_ptr(), p0, p1)


def _mass_stride(mass, name: str, dev: int, B: int, capacity: int) -> int:
    if not isinstance(mass, torch.Tensor) or mass.dtype is not _F32 or mass.shape != (B, capacity) or mass.get_device() != dev:
        _explain(dev, (mass, name, _F32, (B, capacity), False))
    row, one = mass.stride()
    if (one != 1 and capacity > 1) or row < 0:
        raise ValueError(f"{name} rows must be contiguous")
    return row if B > 1 else capacity


def _run(what: str, dev: int, args: bytes) -> None:
    """Call a C entry point on the cache's device and its current stream."""
    fn = getattr(_LIB or _lib(), what)
    if _current_device() == dev:
        rc = fn(args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(args, _raw_stream(dev))
    if rc != 0:
        raise KK3Error(rc, what)


def _workspace(what: str, device: torch.device) -> tuple[torch.Tensor, int]:
    """A call's own workspace, from torch's allocator on the current stream, and its size."""
    nbytes = _WORKSPACE.get((what, device.index))
    if nbytes is None:
        with torch.cuda.device(device):
            nbytes = getattr(_lib(), what)()
        if nbytes <= 0:
            raise KK3Error(-3, what)
        _WORKSPACE[what, device.index] = nbytes
    return torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes


# --- the operators ---------------------------------------------------------------------------------------------

def append(raw, norm_weight, kv, pe, table, lengths, cu_new, *, eps: float = 1e-6, as_step: bool = False,
           error_word=None) -> torch.Tensor:
    """Write the new tokens' entries behind their sequences and return the new lengths (int64 [B]).

    raw: bf16 [T, 576], the `ka` projection of the new tokens; its first 512 values are RMS-normalised with
    norm_weight (bf16 [512]) in FP32 and rounded once, the other 64 are stored as they are. as_step: rounded to bf16
    before the product with norm_weight too, as the model and the decode step do; caches that `step_append` continues
    want this, so that the entry is the one the step would have written. lengths: positions cached before. A token
    behind the table's last column is not written, nor are those of a sequence whose length is negative
    (its new length then counts from zero); both set error_word."""
    cache, dev, B, _ = _cache(kv, pe, table)
    try:
        rs = raw.shape
        fine = (len(rs) == 2 and rs[1] == LATENT + ROPE and raw.dtype is _BF16 and norm_weight.dtype is _BF16
                and norm_weight.shape == (LATENT,) and raw.get_device() == dev and norm_weight.get_device() == dev
                and norm_weight.is_contiguous() and lengths.dtype is _I64 and cu_new.dtype is _I32 and lengths.shape == (B,)
                and cu_new.shape == (B + 1,) and lengths.get_device() == dev and cu_new.get_device() == dev
                and lengths.is_contiguous() and cu_new.is_contiguous())
    except AttributeError:
        fine = False
    if not fine:
        if not isinstance(raw, torch.Tensor) or raw.dim() != 2:
            raise ValueError("raw must be bfloat16 [T, 576]")
        _explain(dev, (raw, "raw", _BF16, (raw.shape[0], LATENT + ROPE), False), (norm_weight, "norm_weight", _BF16, (LATENT,), True),
                 (lengths, "lengths", _I64, (B,), True), (cu_new, "cu_new", _I32, (B + 1,), True))
    T = rs[0]
    row, one = raw.stride()
    if T <= 1:
        row = LATENT + ROPE
    at, weight = raw.data_ptr(), norm_weight.data_ptr()
    if T and (one != 1 or at & 15 or row & 7 or row < LATENT + ROPE) or weight & 15:
        raise ValueError("raw and norm_weight need 16-byte aligned rows with a contiguous last dim")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    out = torch.empty_like(lengths)
    _run("kk3_cache_append_step" if as_step else "kk3_cache_append", dev, _APPEND.pack(
        *cache, at, row, weight, lengths.data_ptr(), cu_new.data_ptr(), out.data_ptr(), _error(error_word, dev), T, eps))
    return out


def attend(q_latent, q_pe, kv, pe, table, lengths, cu_new, *, scale: float | None = None, out=None, lse=None,
           error_word=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of the new tokens over their sequences' caches, in the latent space: (out bf16 [T, heads, 512],
    lse f32 [T, heads]).

    q_latent: bf16 [T, heads, 512] absorbed queries, q_pe: bf16 [T, heads, 64], of any strides (unless
    all (token, head) rows lie at one 16-byte aligned pitch, they are copied first).
    lengths: cached positions, the new tokens included (append's result): token i of n sees the first
    lengths - n + i + 1. A token that sees nothing gets zeros and -inf. Rows behind cu_new[B] are not written (pass
    `out` and `lse`, both contiguous, to keep theirs). What pages hold behind a sequence's length is never used; what
    they hold before it must be finite, also where a token does not see it."""
    cache, dev, B, _ = _cache(kv, pe, table)
    T, H, scale, _keep, q = _queries(q_latent, q_pe, lengths, cu_new, dev, B, scale)
    device = kv.device
    if out is None:
        out = torch.empty_like(q_latent) if q_latent.is_contiguous() else torch.empty(T, H, LATENT, dtype=_BF16, device=device)
    elif out.dtype != _BF16 or out.shape != (T, H, LATENT) or out.get_device() != dev or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"out must be contiguous bfloat16 {[T, H, LATENT]} on the cache's device, 16-byte aligned")
    if lse is None:
        lse = torch.empty(T, H, dtype=_F32, device=device)
    elif lse.dtype != _F32 or lse.shape != (T, H) or lse.get_device() != dev or not lse.is_contiguous():
        raise ValueError(f"lse must be contiguous float32 {[T, H]} on the cache's device")
    err = _error(error_word, dev)
    if T:
        work, nbytes = _workspace("kk3_cache_attend_workspace", device)
        _run("kk3_cache_attend", dev, _ATTEND.pack(*cache, *q, lengths.data_ptr(), cu_new.data_ptr(), out.data_ptr(),
                                                   lse.data_ptr(), work.data_ptr(), nbytes, err, T, H, scale, 0))
    return out, lse


def attention_mass(q_latent, q_pe, lse, kv, pe, table, lengths, cu_new, *, scale: float | None = None, mass=None,
                   out=None, error_word=None) -> torch.Tensor:
    """The attention weight that each cached position gets from the new tokens, summed over tokens and heads and added
    to `mass`: f32 [B, columns * page_size].

    lse: attend's, with the same queries, lengths and scale. mass: what earlier calls accumulated (zeros if None);
    `out` may be mass itself. Positions at or behind a length keep their mass."""
    cache, dev, B, capacity = _cache(kv, pe, table)
    T, H, scale, _keep, q = _queries(q_latent, q_pe, lengths, cu_new, dev, B, scale)
    if not isinstance(lse, torch.Tensor) or lse.dtype is not _F32 or lse.shape != (T, H) or lse.get_device() != dev or not lse.is_contiguous():
        _explain(dev, (lse, "lse", _F32, (T, H), True))
    row, before = 0, 0
    if mass is not None:
        row, before = _mass_stride(mass, "mass", dev, B, capacity), mass.data_ptr()
    device = kv.device
    if out is None:
        out = torch.empty(B, capacity, dtype=_F32, device=device)
    elif out.dtype != _F32 or out.shape != (B, capacity) or out.get_device() != dev or not out.is_contiguous():
        raise ValueError(f"out must be contiguous float32 {[B, capacity]} on the cache's device")
    elif mass is not None and (before != (to := out.data_ptr()) or row != capacity) and to < before + 4 * ((B - 1) * row + capacity) \
            and before < to + 4 * B * capacity:
        raise ValueError("out may be mass itself, but must not overlap it in another way")
    work, nbytes = _workspace("kk3_cache_mass_workspace", device)
    _run("kk3_cache_mass", dev, _MASS.pack(*cache, *q, lse.data_ptr(), lengths.data_ptr(), cu_new.data_ptr(), before, row,
                                           out.data_ptr(), work.data_ptr(), nbytes, _error(error_word, dev), T, H, scale, 0))
    return out


def evict(kv, pe, table, lengths, mass, budget: int, *, sinks: int = 0, recent: int = 0, dst_table=None,
          error_word=None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cut every sequence down to `budget` positions: its first `sinks` and its last `recent` (the lowest of them where
    they are more than the budget), and of the others those of the largest mass (equal ones: the lowest position; NaN
    counts as the largest).

    The kept entries move, in ascending order, to positions 0, 1, ... of dst_table's pages (int32 [B, columns2]; pages
    that none of the sequences uses, so that pages shared with others stay as they are), or in place (None; then no page
    may stand twice in the used part of the table). An entry whose page or new page is outside the pool is counted as
    kept but does not move: its new slot stays as it was, and error_word is set. Returns
    (new lengths int64 [B], their mass f32 [B, columns * page_size] with zeros behind, their old positions int32
    [B, budget] with -1 behind)."""
    cache, dev, B, capacity = _cache(kv, pe, table)
    if (not isinstance(lengths, torch.Tensor) or lengths.dtype is not _I64 or lengths.shape != (B,) or lengths.get_device() != dev
            or not lengths.is_contiguous()):
        _explain(dev, (lengths, "lengths", _I64, (B,), True))
    row = _mass_stride(mass, "mass", dev, B, capacity)
    budget, sinks, recent = int(budget), int(sinks), int(recent)
    if not 1 <= budget <= capacity:
        raise ValueError("budget must be 1 .. columns * page_size")
    if not 0 <= sinks <= MAX_POSITIONS or not 0 <= recent <= MAX_POSITIONS:
        raise ValueError(f"sinks and recent must be 0 .. {MAX_POSITIONS}")
    dst, dst_row, dst_columns = 0, 0, 0
    if dst_table is not None:
        if not isinstance(dst_table, torch.Tensor) or dst_table.dim() != 2:
            raise ValueError("dst_table must be int32 [B, columns]")
        dst_columns = dst_table.shape[1]
        if dst_table.dtype is not _I32 or dst_table.shape[0] != B or dst_table.get_device() != dev:
            _explain(dev, (dst_table, "dst_table", _I32, (B, dst_columns), False))
        dst_row, one = dst_table.stride()
        if (one != 1 and dst_columns > 1) or dst_row < 0:
            raise ValueError("dst_table rows must be contiguous")
        if dst_columns * kv.shape[1] < budget:
            raise ValueError("dst_table must hold the budget")
        dst, dst_row = dst_table.data_ptr(), dst_row if B > 1 else dst_columns
    device = kv.device
    new_lengths = torch.empty_like(lengths)
    new_mass = torch.empty(B, capacity, dtype=_F32, device=device)
    kept = torch.empty(B, budget, dtype=_I32, device=device)
    _run("kk3_cache_evict", dev, _EVICT.pack(*cache, lengths.data_ptr(), mass.data_ptr(), row, dst, dst_row,
                                             new_lengths.data_ptr(), new_mass.data_ptr(), kept.data_ptr(),
                                             _error(error_word, dev), budget, sinks, recent, dst_columns))
    return new_lengths, new_mass, kept
