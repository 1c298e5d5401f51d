"""CPU tests of the cache operators' C ABI (include/pmkl_cache.h): layouts, what each call refuses before any launch, and
the 64-bit reference that the GPU tests compare with."""
from __future__ import annotations

import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

from pmkl_amd import capi
from tests import cache_reference as ref

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "pmkl_cache.h"


def test_header_declares_the_exported_set():
    names = set(re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(pmkl_\w+)\s*\(", HEADER.read_text(), re.M))
    assert names == set(capi.CACHE_SYMBOLS)
    lib = capi.load()
    for name in names:
        assert hasattr(lib, name), name


@pytest.mark.parametrize("cname,cls", [("pmkl_kv_cache", "KvCache"), ("pmkl_cache_slots_args", "CacheSlotsArgs"),
                                       ("pmkl_cache_append_args", "CacheAppendArgs"),
                                       ("pmkl_cache_attn_args", "CacheAttnArgs")])
def test_struct_layout_matches_header(tmp_path, cname, cls):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    mirror = getattr(capi, cls)
    fields = [f[0] for f in mirror._fields_]
    body = "".join(f'  printf("{f} %zu\\n", offsetof({cname}, {f}));\n' for f in fields)
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "pmkl_cache.h"\nint main(void) {\n' + body +
                   f'  printf("sizeof %zu\\n", sizeof({cname}));\n  return 0;\n}}\n')
    subprocess.run([cc, "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    out = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True,
                                                         check=True).stdout.splitlines())
    for f in fields:
        assert int(out[f]) == getattr(mirror, f).offset, f
    assert int(out["sizeof"]) == ctypes.sizeof(mirror)


def _refused(rc, code, pattern):
    msg = capi.last_error()
    assert rc == code, (rc, msg)
    assert re.search(pattern, msg), msg
    assert re.search(r"pmkl check failed at cache_capi\.hip:\d+", msg), msg


def _cache(**kw):
    base = dict(k=0x10000, v=0x20000, k_scale=0x30000, v_scale=0x40000, pages=8, kv_heads=2, page_size=16, head_dim=64)
    base.update(kw)
    return capi.make_kv_cache(**base)


def _slots(**kw):
    base = dict(cached_lens=0x1000, new_lens=0x2000, block_table=0x3000, free_pages=0x4000, free_head=0x5000,
                seq_lens=0x6000, query_start=0x7000, slots=0x8000, free_head_out=0x9000, batch=4, table_width=8,
                free_count=16, page_size=16, tokens=4)
    base.update(kw)
    return capi.cache_slots_raw(capi.make_cache_slots_args(**base))


def _append(cache=None, **kw):
    base = dict(k=0x50000, v=0x60000, slots=0x70000, dtype=capi.PMKL_DTYPE_BF16, tokens=4)
    base.update(kw)
    return capi.cache_append_raw(capi.make_cache_append_args(_cache(**(cache or {})), **base))


def _attn_args(cache=None, **kw):
    base = dict(q=0x50000, o=0x60000, m=0x70000, l=0x71000, block_table=0x72000, seq_lens=0x73000, query_start=0x74000,
                workspace=0x100000, workspace_bytes=1 << 40, dtype=capi.PMKL_DTYPE_BF16, is_causal=1, tokens=4, heads=4,
                batch=4, table_width=8)
    base.update(kw)
    return capi.make_cache_attn_args(_cache(**(cache or {})), **base)


def _attn(cache=None, **kw):
    return capi.cache_attn_fwd_raw(_attn_args(cache, **kw))


def test_null_arguments():
    lib = capi.load()
    for name in ("pmkl_cache_slots", "pmkl_cache_append", "pmkl_cache_attn_fwd"):
        _refused(getattr(lib, name)(None, None), capi.PMKL_EINVAL, "args is a null pointer")
    assert lib.pmkl_cache_attn_workspace_size(None) == 0
    assert lib.pmkl_cache_attn_kernel_name(None) is None


@pytest.mark.parametrize("page_size", [0, 8, 24, 512, -16])
def test_page_sizes_refused(page_size):
    for rc in (_slots(page_size=page_size), _append({"page_size": page_size}), _attn({"page_size": page_size})):
        _refused(rc, capi.PMKL_EINVAL, "power of two from 16 to 256")


@pytest.mark.parametrize("kw,pattern", [
    (dict(batch=-1), "batch -1"), (dict(tokens=1 << 31), "tokens 2147483648"), (dict(table_width=-2), "table_width -2"),
    (dict(free_count=1 << 31), "free_count"), (dict(table_stride=7), "table_stride 7 < table_width 8"),
    (dict(cached_lens=0), "cached_lens is a null"), (dict(new_lens=0), "new_lens is a null"),
    (dict(block_table=0), "block_table is a null"), (dict(free_pages=0), "free_pages is a null"),
    (dict(free_head=0), "free_head is a null"), (dict(seq_lens=0x6002), "seq_lens must be 4-byte aligned"),
    (dict(slots=0x8004), "slots must be 8-byte aligned"), (dict(query_start=0), "query_start is a null"),
    (dict(free_head_out=0), "free_head_out is a null"),
    # outputs on inputs, or on each other
    (dict(seq_lens=0x1000), "seq_lens overlaps cached_lens"), (dict(seq_lens=0x2008), "seq_lens overlaps new_lens"),
    (dict(free_head_out=0x5000), "free_head_out overlaps free_head"), (dict(free_pages=0x3040), "block_table overlaps free_pages"),
    (dict(query_start=0x5ffc), "query_start overlaps seq_lens"), (dict(slots=0x7010), "slots overlaps query_start"),
])
def test_slots_refusals(kw, pattern):
    _refused(_slots(**kw), capi.PMKL_EINVAL, pattern)


CACHE_REFUSALS = [
    (dict(pages=-1), capi.PMKL_EINVAL, "pages -1"), (dict(pages=1 << 31), capi.PMKL_EINVAL, "pages 2147483648"),
    (dict(pages=0), capi.PMKL_EINVAL, "no pages"),
    (dict(head_dim=80), capi.PMKL_EUNSUPPORTED, "head_dim 80"), (dict(head_dim=256), capi.PMKL_EUNSUPPORTED, "head_dim 256"),
    (dict(kv_heads=0), capi.PMKL_EINVAL, "kv_heads 0"),
    (dict(k=0), capi.PMKL_EINVAL, "k_cache is a null"), (dict(v=0x20008), capi.PMKL_EINVAL, "v_cache must be 16-byte"),
    (dict(k_scale=0), capi.PMKL_EINVAL, "k_scale is a null"), (dict(v_scale=0x40002), capi.PMKL_EINVAL, "v_scale must be 4-byte"),
    (dict(k_strides=(2048, 1024, 72)), capi.PMKL_EINVAL, "k_cache stride 72 must be a non-negative multiple of 16"),
    (dict(v_strides=(-2048, 1024, 16)), capi.PMKL_EINVAL, "v_cache stride -2048"),
    (dict(k_strides=(1 << 33, 1 << 32, 1 << 31)), capi.PMKL_EINVAL, "more than 2 GiB"),
    (dict(k_strides=(1 << 62, 1024, 64)), capi.PMKL_EINVAL, "span too many"),
    (dict(k_scale_strides=(-2, 1)), capi.PMKL_EINVAL, "k_scale stride -2"),
]
OVERLAPS = [
    (dict(k_strides=(1024, 1024, 64)), "k_cache strides make distinct rows overlap"),
    (dict(v_strides=(2048, 1024, 0)), "v_cache strides make"), (dict(k_scale_strides=(0, 1)), "k_scale strides make"),
    (dict(v_scale_strides=(1, 1)), "v_scale strides make"),
]


@pytest.mark.parametrize("kw,code,pattern", CACHE_REFUSALS)
def test_cache_refusals(kw, code, pattern):
    if "kv_heads" in kw:
        _refused(_append(kw), code, pattern)
    else:
        _refused(_append(kw), code, pattern)
        _refused(_attn(kw), code, pattern)


@pytest.mark.parametrize("kw,pattern", OVERLAPS)
def test_append_refuses_a_cache_that_overlaps_itself(kw, pattern):
    _refused(_append(kw), capi.PMKL_EINVAL, pattern)


@pytest.mark.parametrize("kw,code,pattern", [
    (dict(dtype=7), capi.PMKL_EUNSUPPORTED, "unsupported dtype 7"), (dict(tokens=-1), capi.PMKL_EINVAL, "tokens -1"),
    (dict(k=0), capi.PMKL_EINVAL, "k is a null"), (dict(v=0x60008), capi.PMKL_EINVAL, "v must be 16-byte"),
    (dict(slots=0), capi.PMKL_EINVAL, "slots is a null"),
    (dict(k_strides=(128, 68)), capi.PMKL_EINVAL, "k stride 68 must be a non-negative multiple of 8"),
    (dict(v_strides=(-128, 64)), capi.PMKL_EINVAL, "v stride -128"),
])
def test_append_refusals(kw, code, pattern):
    _refused(_append(**kw), code, pattern)


@pytest.mark.parametrize("kw,code,pattern", [
    (dict(dtype=7), capi.PMKL_EUNSUPPORTED, "unsupported dtype 7"), (dict(tokens=-1), capi.PMKL_EINVAL, "not negative"),
    (dict(heads=5), capi.PMKL_EINVAL, "heads 5 is not a multiple of kv_heads 2"),
    (dict(scale=float("nan")), capi.PMKL_EINVAL, "scale"), (dict(scale=-1.0), capi.PMKL_EINVAL, "scale"),
    (dict(batch=-1), capi.PMKL_EINVAL, "batch -1"), (dict(table_width=1 << 31), capi.PMKL_EINVAL, "table_width"),
    (dict(tokens=1 << 30), capi.PMKL_EINVAL, "past 2"), (dict(table_width=1 << 27), capi.PMKL_EINVAL, "past 2.31 tokens"), (dict(table_stride=-8), capi.PMKL_EINVAL, "table_stride -8"),
    (dict(q=0), capi.PMKL_EINVAL, "q is a null"), (dict(o=0x60004), capi.PMKL_EINVAL, "o must be 16-byte"),
    (dict(m=0), capi.PMKL_EINVAL, "m is a null"), (dict(l=0x71001), capi.PMKL_EINVAL, "l must be 4-byte"),
    (dict(block_table=0), capi.PMKL_EINVAL, "block_table is a null"), (dict(seq_lens=0), capi.PMKL_EINVAL, "seq_lens is"),
    (dict(query_start=0), capi.PMKL_EINVAL, "query_start is a null"),
    (dict(q_strides=(256, 60)), capi.PMKL_EINVAL, "q stride 60"),
    (dict(o_strides=(64, 64)), capi.PMKL_EINVAL, "o strides make distinct rows overlap"),
])
def test_attn_refusals(kw, code, pattern):
    _refused(_attn(**kw), code, pattern)


def test_nothing_to_do_succeeds_without_touching_anything():
    assert _append(dict(k=0, v=0, k_scale=0, v_scale=0), k=0, v=0, slots=0, tokens=0) == capi.PMKL_OK
    for kw in (dict(tokens=0), dict(batch=0), dict(heads=0)):
        args = _attn_args(dict(k=0, v=0, k_scale=0, v_scale=0, pages=0), q=0, o=0, m=0, l=0, workspace=0, **kw)
        assert capi.cache_attn_fwd_raw(args) == capi.PMKL_OK
        assert capi.cache_attn_kernel_name(args) == "none"
        assert capi.load().pmkl_cache_attn_workspace_size(ctypes.byref(args)) == 0


def test_torch_entry_points_refuse_host_tensors():
    import torch

    import pmkl_amd

    x = torch.zeros(1, 1, 32)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm device tensors"):
        pmkl_amd.cache_slots(i, i, i[None], i, i, 16, 1)
    with pytest.raises(RuntimeError, match="ROCm device tensors"):
        pmkl_amd.cache_append(x, x, i.long(), x, x, x, x)
    with pytest.raises(RuntimeError, match="ROCm device tensors"):
        pmkl_amd.cache_attn_fwd(x, x, x, x, x, i[None], i, i)


def test_reference_encoder_is_torchs():
    """encode() against torch's conversion to float8_e4m3fn on the CPU, with ties and subnormals among the values."""
    import torch

    grid = np.concatenate([ref.E4M3[:127], (ref.E4M3[:126] + ref.E4M3[1:127]) / 2])
    x = np.concatenate([grid, -grid, np.random.default_rng(0).normal(size=5000) * 40, [np.nan]]).clip(-448, 448)
    codes = torch.from_numpy(x).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    x32 = torch.from_numpy(x).float().double().numpy()
    assert np.array_equal(ref.encode(x32) & np.where(np.isnan(x32), 0x7f, 0xff), codes & np.where(np.isnan(x32), 0x7f, 0xff))
    assert np.array_equal(ref.E4M3[:127], torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy())


def test_reference_scale():
    for a in (0.0, 1e-45, 1.0, 448.0, np.nextafter(np.float32(448), np.float32(1e9)), 3.4e38):
        s = ref.need(float(a))
        assert a <= 448 * s and (s == 2.0 ** -126 or a > 448 * s / 2)
