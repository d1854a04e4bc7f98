"""The paged latent cache's argument checks (kimi_k3_goalbox_b200/latent_cache.py, include/kk3.h): what a call refuses is
refused on the host, before anything is enqueued, so these need no GPU."""

from __future__ import annotations

import ctypes
import shutil
import struct
import subprocess
from pathlib import Path

import pytest
import torch

from kimi_k3_goalbox_b200 import latent_cache as lc
from kimi_k3_goalbox_b200.runtime import load_library

ROOT = Path(__file__).resolve().parents[1]
BF, F32, I32, I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64
OK, ERR_ARG, ERR_UNSUPPORTED, ERR_CUDA = 0, -1, -2, -3


def test_paged_view_addresses_the_same_entries():
    kv, pe = torch.arange(2 * 12 * 512, dtype=F32).view(2, 12, 512), torch.zeros(2, 12, 64)
    pages, rope, table = lc.paged_view(kv, pe, 4)
    assert table.dtype == I32 and table.tolist() == [[0, 1, 2], [3, 4, 5]] and rope.shape == (6, 4, 64)
    for b in range(2):
        for p in range(12):
            assert torch.equal(pages[table[b, p // 4], p % 4], kv[b, p])
    pages[4, 1] = -1.0
    assert bool((kv[1, 5] == -1).all())
    for page in (5, 0, -4):
        with pytest.raises(ValueError):
            lc.paged_view(kv, pe, page)
    with pytest.raises(ValueError):
        lc.paged_view(kv, pe[:, :8], 4)


def _call(op, **change):
    """An operator on host tensors with some arguments changed."""
    B, T, H, page, columns = 2, 3, 4, 16, 2
    a = {"kv": torch.zeros(5, page, 512, dtype=BF), "pe": torch.zeros(5, page, 64, dtype=BF), "table": torch.zeros(B, columns, dtype=I32),
         "lengths": torch.zeros(B, dtype=I64), "cu_new": torch.zeros(B + 1, dtype=I32), "raw": torch.zeros(T, 576, dtype=BF),
         "norm_weight": torch.zeros(512, dtype=BF), "q_latent": torch.zeros(T, H, 512, dtype=BF), "q_pe": torch.zeros(T, H, 64, dtype=BF),
         "lse": torch.zeros(T, H), "mass": torch.zeros(B, page * columns), "budget": 8}
    takes = {"append": ("raw", "norm_weight", "kv", "pe", "table", "lengths", "cu_new"),
             "attend": ("q_latent", "q_pe", "kv", "pe", "table", "lengths", "cu_new"),
             "attention_mass": ("q_latent", "q_pe", "lse", "kv", "pe", "table", "lengths", "cu_new"),
             "evict": ("kv", "pe", "table", "lengths", "mass", "budget")}[op]
    named = {k: v for k, v in change.items() if k not in takes}
    a.update(change)
    return getattr(lc, op)(*(a[k] for k in takes), **named)


@pytest.mark.parametrize("op", ["append", "attend", "attention_mass", "evict"])
@pytest.mark.parametrize("change,message", [
    ({}, "CUDA device"),
    ({"kv": None}, "kv must be a tensor"),
    ({"kv": torch.zeros(5, 16, 512)}, "kv must be torch.bfloat16"),
    ({"kv": torch.zeros(5, 16, 511, dtype=BF)}, "kv must be"),
    ({"kv": torch.zeros(0, 16, 512, dtype=BF)}, "not empty"),
    ({"pe": torch.zeros(5, 8, 64, dtype=BF)}, "pe must be"),
    ({"pe": torch.zeros(5, 16, dtype=BF)}, "pe must be a tensor of 3 dims"),
    ({"table": torch.zeros(2, 2, dtype=I64)}, "table must be torch.int32"),
    ({"table": torch.zeros(2, 0, dtype=I32)}, "not empty"),
])
def test_caches_that_do_not_fit_are_refused(op, change, message):
    with pytest.raises(ValueError, match=message):
        _call(op, **change)


def _entry(name):
    fn = getattr(load_library(), name)
    fn.argtypes, fn.restype = [ctypes.c_char_p, ctypes.c_void_p], ctypes.c_int
    return fn


P = 1 << 20     # an address that nothing reads: every call below is refused before its launch
CACHE = dict(kv=P, pe=P, kv_page=16 * 512, kv_row=512, pe_page=16 * 64, pe_row=64, table=P, table_stride=4, num_pages=8, page_size=16,
             columns=4, batch=2)
APPEND = dict(raw=P, raw_stride=576, norm_weight=P, lengths=P, cu_new=P, new_lengths=2 * P, error_word=0, tokens=3, eps=1e-6)
ATTEND = dict(q_latent=P, ql_token=2048, ql_head=512, q_pe=P, qp_token=256, qp_head=64, lengths=P, cu_new=P, out=P, lse=P, workspace=P,
              workspace_bytes=1 << 40, error_word=0, tokens=3, heads=4, scale=0.1, pad=0)
MASS = dict(q_latent=P, ql_token=2048, ql_head=512, q_pe=P, qp_token=256, qp_head=64, lse=P, lengths=P, cu_new=P, mass=0, mass_stride=64,
            new_mass=P, workspace=P, workspace_bytes=1 << 40, error_word=0, tokens=3, heads=4, scale=0.1, pad=0)
EVICT = dict(lengths=P, mass=P, mass_stride=64, dst_table=0, dst_stride=0, new_lengths=2 * P, new_mass=2 * P, kept=P, error_word=0, budget=8,
             sinks=0, recent=0, dst_columns=0)
BLOCKS = {"append": (lc._APPEND, APPEND), "attend": (lc._ATTEND, ATTEND), "mass": (lc._MASS, MASS), "evict": (lc._EVICT, EVICT)}


def _refusal(op, **change):
    layout, fields = BLOCKS[op]
    both = CACHE | fields
    assert change.keys() <= both.keys()
    values = list((CACHE | {k: v for k, v in change.items() if k in CACHE}).values()) + list(
        (fields | {k: v for k, v in change.items() if k in fields}).values())
    return _entry(f"kk3_cache_{op}")(layout.pack(*values), None)


@pytest.mark.parametrize("op", list(BLOCKS))
@pytest.mark.parametrize("change", [
    {"kv": 0}, {"pe": 0}, {"table": 0}, {"kv": P + 8}, {"pe": P + 2}, {"table": P + 2}, {"num_pages": 0}, {"page_size": 0}, {"columns": 0},
    {"batch": 0}, {"batch": -1}, {"num_pages": -3}, {"kv_row": 508}, {"pe_row": 60}, {"kv_page": -8192}, {"table_stride": -1},
    {"batch": 4097}, {"page_size": 65537}, {"columns": 1 << 24}, {"lengths": 0}, {"lengths": P + 4}])
def test_entry_points_refuse_bad_caches(op, change):
    assert _refusal(op, **change) in (ERR_ARG, ERR_UNSUPPORTED)


@pytest.mark.parametrize("op,change", [
    *[("append", c) for c in ({"raw": 0}, {"raw": P + 2}, {"raw_stride": 575}, {"raw_stride": 568}, {"norm_weight": 0}, {"cu_new": 0},
                              {"new_lengths": 0}, {"tokens": -1}, {"eps": -1.0}, {"eps": float("nan")})],
    *[(op, c) for op in ("attend", "mass") for c in (
        {"q_latent": 0}, {"q_latent": P + 2}, {"q_pe": P + 8}, {"ql_token": 2044}, {"qp_head": 60}, {"ql_head": -512}, {"lse": 0},
        {"cu_new": 0}, {"tokens": -1}, {"heads": 0}, {"heads": 129}, {"scale": float("nan")}, {"tokens": 1 << 30})],
    ("attend", {"out": 0}), ("attend", {"out": P + 8}), ("mass", {"new_mass": 0}), ("mass", {"mass": P + 2}), ("mass", {"mass_stride": -1, "mass": P}),
    *[("evict", c) for c in ({"mass": 0}, {"mass_stride": -1}, {"budget": 0}, {"budget": 65}, {"sinks": -1}, {"recent": -1},
                             {"kept": 0}, {"new_mass": 0}, {"new_lengths": 0}, {"new_mass": P}, {"new_lengths": P},
                             {"dst_table": P + 2}, {"dst_table": P, "dst_columns": 0}, {"dst_table": P, "dst_columns": 4, "dst_stride": -4})]])
def test_entry_points_refuse_bad_arguments(op, change):
    assert _refusal(op, **change) in (ERR_ARG, ERR_UNSUPPORTED)


@pytest.mark.parametrize("op", list(BLOCKS))
def test_entry_points_refuse_no_arguments(op):
    assert _entry(f"kk3_cache_{op}")(None, None) == ERR_ARG
    assert _entry(f"kk3_cache_{op}")(bytes(BLOCKS[op][0].size), None) == ERR_ARG


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler")
def test_argument_blocks_match_the_header(tmp_path):
    names = [f"kk3_cache_{op}_args" for op in BLOCKS]
    body = "".join(f'printf("%zu\\n", sizeof({n}));' for n in names)
    (tmp_path / "s.c").write_text(f'#include <stdio.h>\n#include "kk3.h"\nint main(void) {{ {body} return 0; }}\n')
    subprocess.run(["gcc", "-I", str(ROOT / "include"), "-o", str(tmp_path / "s"), str(tmp_path / "s.c")], check=True)
    sizes = [int(v) for v in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    assert sizes == [layout.size for layout, _ in BLOCKS.values()]
    assert struct.calcsize("=" + lc._CACHE) == sizes[0] - struct.calcsize("=QqQQQQQif")


@pytest.mark.parametrize("stride", [0, 32, 63, 65, 128])
def test_mass_in_place_needs_the_stride_of_the_result(stride):
    assert _refusal("mass", mass=P, new_mass=P, mass_stride=stride) == ERR_ARG


@pytest.mark.parametrize("op", ["attend", "mass"])
@pytest.mark.parametrize("scale", [2.4e38, -3e38, float("inf"), -float("inf"), float("nan")])
def test_entry_points_refuse_scales_that_leave_fp32(op, scale):
    assert _refusal(op, scale=scale) == ERR_ARG
