"""CPU tier of the paged-cache entry points: the kernels' index arithmetic, and what the calls refuse before they touch
the device."""
import ctypes as ct
import os
import subprocess

import numpy as np
import pytest

from conftest import ROOT

CPP = os.path.join(ROOT, "tests", "cpp")


def test_index_arithmetic():
    subprocess.run(["make", "-s", "-C", CPP, "paged_index_check"], check=True)
    assert subprocess.run([os.path.join(CPP, "paged_index_check")], check=True, capture_output=True, text=True).stdout == "ok\n"


BUF = np.zeros(4096 + 64, dtype=np.uint8)  # never touched: every call here is refused
BASE = (BUF.ctypes.data + 63) // 64 * 64


def at(offset=0):
    return BASE + offset


def cache_struct(fa, **change):
    a = dict(k=at(), v=at(), k_strides=(2048, 1024, 64), v_strides=(2048, 1024, 64), n_pages=2, page_size=16, heads=2, head_dim=64)
    a.update(change)
    return fa._PagedCacheStruct(a["k"], a["v"], (ct.c_int64 * 3)(*a["k_strides"]), (ct.c_int64 * 3)(*a["v_strides"]),
                                a["n_pages"], a["page_size"], a["heads"], a["head_dim"])


def plan(fa, **change):
    a = dict(k_len=at(), n_new=at(256), table=at(512), stride=4, free=at(1024), free_count=at(1280), q_start=at(1536), k_out=at(1792),
             slots=at(2048), counts=at(2304), B=2, width=4, page=16, cap=8, tokens=8)
    a.update(change)
    return fa.lib().fa_cache_plan(*[a[k] for k in ("k_len", "n_new", "table", "stride", "free", "free_count", "q_start", "k_out", "slots",
                                                   "counts", "B", "width", "page", "cap", "tokens")], None, None)


@pytest.mark.parametrize("change,status", [
    (dict(page=8), 4), (dict(page=24), 4), (dict(page=0), 4), (dict(page=1 << 17), 4), (dict(B=0), 4), (dict(B=5121), 4),
    (dict(width=0), 4), (dict(width=1 << 27, stride=1 << 27), 4), (dict(stride=3), 4), (dict(cap=-1), 4), (dict(tokens=-1), 4),
    (dict(k_len=None), 5), (dict(n_new=None), 5), (dict(table=None), 5), (dict(free=None), 5), (dict(free_count=None), 5),
    (dict(q_start=None), 5), (dict(k_out=None), 5), (dict(slots=None), 5), (dict(counts=None), 5),
    (dict(k_out=at()), 5), (dict(counts=at(1280)), 5), (dict(q_start=at(260)), 5), (dict(slots=at(4)), 5),
])
def test_plan_refusals(fa, change, status):
    assert plan(fa, **change) == status
    assert b"fa_cache_plan" in fa.lib().fa_last_error()


CACHE_REFUSALS = [
    (dict(k=None), 5), (dict(v=None), 5), (dict(head_dim=96), 3), (dict(head_dim=0), 3), (dict(heads=0), 4), (dict(n_pages=0), 4),
    (dict(page_size=8), 4), (dict(page_size=48), 4), (dict(k=at(8)), 4), (dict(v=at(2)), 4), (dict(k_strides=(2048, 1024, 60)), 4),
    (dict(v_strides=(2048, -1024, 64)), 4), (dict(k_strides=(2048, 1024, 56)), 4), (dict(k_strides=(2048, 1024, 1 << 26)), 4),
]


def write(fa, cache, **change):
    a = dict(k=at(), v=at(), k_tok=128, k_head=64, v_tok=128, v_head=64, slots=at(512), tokens=1)
    a.update(change)
    return fa.lib().fa_cache_write(a["k"], a["v"], a["k_tok"], a["k_head"], a["v_tok"], a["v_head"], ct.byref(cache), a["slots"], a["tokens"], None, None)


@pytest.mark.parametrize("change,status", CACHE_REFUSALS)
def test_cache_refusals(fa, change, status):
    c = cache_struct(fa, **change)
    assert write(fa, c) == status
    assert shared(fa, c) == status


@pytest.mark.parametrize("change,status", [
    (dict(k=None), 5), (dict(v=None), 5), (dict(slots=None), 5), (dict(tokens=-1), 4), (dict(tokens=1 << 30), 4), (dict(k=at(8)), 4),
    (dict(k_tok=4), 4), (dict(v_head=-64), 4),
])
def test_write_refusals(fa, change, status):
    assert write(fa, cache_struct(fa), **change) == status


def test_calls_that_would_not_fit_a_launch(fa):
    wide = dict(heads=4096, k_strides=(ct.c_int64 * 3)(1 << 22, 64 * 16, 64), v_strides=(ct.c_int64 * 3)(1 << 22, 64 * 16, 64))
    assert write(fa, cache_struct(fa, **wide), tokens=1 << 17) == 4


def test_output_over_the_queries_is_refused(fa):
    assert shared(fa, cache_struct(fa), o=at(), ws_bytes=1 << 40) == 5


def test_calls_without_work_report_no_time(fa):
    L, ms = fa.lib(), ct.c_float(7.0)
    assert L.fa_cache_write(None, None, 64, 64, 64, 64, ct.byref(cache_struct(fa)), None, 0, None, ct.byref(ms)) == 0 and ms.value == 0.0
    ms = ct.c_float(7.0)
    assert L.fa_forward_shared_prefix(None, 64, 64, None, 64, 64, ct.byref(cache_struct(fa)), None, 0, None, 0, 0, None, None, 0, 1, 4, 0, 1,
                                      0.125, 0, None, 0, None, ct.byref(ms)) == 0 and ms.value == 0.0


def test_nothing_to_write_is_no_error(fa):
    assert write(fa, cache_struct(fa), tokens=0, k=None, v=None) == 0


def shared(fa, cache, **change):
    a = dict(q=at(), q_tok=256, q_head=64, o=at(1024), o_tok=256, o_head=64, prefix=at(), prefix_len=16, table=at(), stride=4, width=4,
             q_start=at(), k_len=at(), T=1, B=1, Hq=4, dtype=0, flags=1, scale=0.125, max_k=64, ws=at(), ws_bytes=0)
    a.update(change)
    return fa.lib().fa_forward_shared_prefix(
        a["q"], a["q_tok"], a["q_head"], a["o"], a["o_tok"], a["o_head"], ct.byref(cache) if cache is not None else None, a["prefix"],
        a["prefix_len"], a["table"], a["stride"], a["width"], a["q_start"], a["k_len"], a["T"], a["B"], a["Hq"], a["dtype"], a["flags"],
        a["scale"], a["max_k"], a["ws"], a["ws_bytes"], None, None)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), 4), (dict(flags=2), 4), (dict(scale=float("nan")), 4), (dict(scale=float("inf")), 4), (dict(scale=0.0), 4), (dict(scale=-0.1), 4),
    (dict(scale=1e-40), 4), (dict(T=-1), 4), (dict(B=-1), 4),
    (dict(Hq=3), 4), (dict(Hq=0), 4), (dict(prefix_len=-1), 2), (dict(prefix_len=(1 << 30) + 1), 2), (dict(max_k=-1), 2),
    (dict(T=1 << 24, Hq=4), 4), (dict(B=4001), 4), (dict(Hq=258), 4), (dict(width=-1), 4), (dict(stride=3), 4), (dict(width=1 << 27, stride=1 << 27), 4), (dict(q=None), 5),
    (dict(o=None), 5), (dict(prefix=None), 5), (dict(table=None), 5), (dict(q_start=None), 5), (dict(k_len=None), 5), (dict(q=at(8)), 4),
    (dict(o_tok=-256), 4), (dict(q_head=60), 4), (dict(), 7), (dict(ws=None, ws_bytes=1 << 40), 7), (dict(ws=at(8), ws_bytes=1 << 40), 7),
])
def test_shared_prefix_refusals(fa, change, status):
    assert shared(fa, cache_struct(fa), **change) == status
    assert fa.lib().fa_last_error()


def test_shared_prefix_without_rows_is_no_error(fa):
    assert shared(fa, cache_struct(fa), T=0) == 0
    assert shared(fa, cache_struct(fa), B=0) == 0
    assert shared(fa, None) == 5


def test_workspace_of_refused_sizes_is_none(fa):
    L = fa.lib()
    assert L.fa_shared_prefix_workspace(1, 1, 4, 3, 64, 0, 16) == 0
    assert L.fa_shared_prefix_workspace(0, 1, 4, 2, 64, 0, 16) == 0
    assert L.fa_shared_prefix_workspace(1, 1, 4, 2, 64, -1, 16) == 0
    assert L.fa_shared_prefix_workspace(1, 4001, 4, 2, 64, 0, 16) == 0
    assert L.fa_shared_prefix_workspace(1, 1, 129, 1, 64, 0, 16) == 0
    assert L.fa_shared_prefix_workspace(1, 1, 4, 2, 96, 0, 16) == 0
    assert L.fa_shared_prefix_workspace(1, 1, 4, 2, 64, 0, 16) >= 4 * (64 + 2) * 4


def test_workspace_of_many_rows_is_bounded(fa):
    """1 GiB, or three parts (a prefix' and two of a request's own keys) and a count a row."""
    for T, B, Hq, Hkv, D, prefix in [(65536, 1, 64, 8, 128, 0), (4096, 1, 32, 8, 128, 8192), (8000, 8, 32, 8, 128, 8192), (20000, 2, 32, 4, 64, 0),
                                     (100000, 4, 16, 2, 256, 100), (1, 1, 128, 1, 256, 1 << 20), (512, 512, 64, 8, 128, 1 << 20)]:
        rows = T * Hq
        assert fa.lib().fa_shared_prefix_workspace(T, B, Hq, Hkv, D, prefix, 1 << 20) <= max(1 << 30, 3 * rows * (D + 2) * 4) + 4 * rows


def test_python_refusals(fa):
    import torch

    with pytest.raises(ValueError):
        fa.PagedCache(torch.zeros(1, 1, 16, 64, dtype=torch.float16), torch.zeros(1, 1, 16, 64, dtype=torch.float16))
    z = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(fa.FlashAttentionError):
        fa.cache_plan(z, z, z[None], z, z, 16, 4)
