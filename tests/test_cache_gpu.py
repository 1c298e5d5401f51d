"""GPU tests of the cache operators against their 64-bit definitions (tests/cache_reference.py, whose bounds count the
roundings): sizes and masks where they can go wrong, what they must leave alone, streams and graphs, and a serving run of
all three."""
from __future__ import annotations

import math
import sys

import numpy as np
import pytest

from tests import cache_reference as ref

pytestmark = pytest.mark.gpu


def _say(msg):
    print(msg, flush=True)
    sys.stdout.flush()


def _dtype(name):
    from pmkl_amd.workloads import torch_dtype

    return torch_dtype(name)


def _np(t):
    return t.detach().cpu().double().numpy()


def _codes(t):
    import torch

    return t.view(torch.uint8).cpu().numpy()


def _int32(values):
    import torch

    return torch.tensor(values, dtype=torch.int32, device="cuda:0")


class Cache:
    """Tensors of a cache and its requests' table.  Every page holds NaN codes, under scales of NaN, until it is filled:
    what a kernel must not read into a result shows."""

    def __init__(self, lengths, kv_heads, page, dim, seed, spare=3, width_more=1, interleaved=False):
        import torch

        rng = np.random.default_rng(seed)
        counts = [-(-n // page) for n in lengths]
        pages = sum(counts) + spare
        order = rng.permutation(pages)
        self.table = np.full((len(lengths), max(counts, default=0) + width_more), -1, dtype=np.int64)
        k = np.full((pages, kv_heads, page, dim), 0x7f, dtype=np.uint8)
        v = np.full((pages, kv_heads, dim, page), 0xff, dtype=np.uint8)
        ks, vs = (np.full((pages, kv_heads), np.nan, dtype=np.float32) for _ in range(2))
        at = 0
        for b, n in enumerate(lengths):
            for w in range(counts[b]):
                p = int(order[at])
                at += 1
                self.table[b, w] = p
                ks[p], vs[p] = (rng.uniform(0.5, 2, kv_heads).astype(np.float32) * 2.0 ** rng.integers(-9, -5) for _ in range(2))
                fill = min(page, n - w * page)
                k[p, :, :fill] = ref.encode(rng.normal(size=(kv_heads, fill, dim)).clip(-4, 4) * 100)
                v[p, :, :, :fill] = ref.encode(rng.normal(size=(kv_heads, dim, fill)).clip(-4, 4) * 100)
        self.k, self.v, self.k_scale, self.v_scale = k, v, ks, vs
        self.lengths = list(lengths)
        if interleaved:   # heads innermost, as the rows of a projection lie
            kt = torch.from_numpy(k.transpose(0, 2, 1, 3).copy()).to("cuda:0").permute(0, 2, 1, 3)
            vt = torch.from_numpy(v.transpose(0, 2, 1, 3).copy()).to("cuda:0").permute(0, 2, 1, 3)
        else:
            kt, vt = torch.from_numpy(k).to("cuda:0"), torch.from_numpy(v).to("cuda:0")
        self.tensors = {"k_cache": kt.view(torch.float8_e4m3fn), "v_cache": vt.view(torch.float8_e4m3fn),
                        "k_scale": torch.from_numpy(ks).to("cuda:0"), "v_scale": torch.from_numpy(vs).to("cuda:0")}

    def refresh(self):
        """Takes the tensors over after a change of the host arrays."""
        import torch

        for name, a in (("k_cache", self.k), ("v_cache", self.v)):
            self.tensors[name].view(torch.uint8).copy_(torch.from_numpy(a))
        self.tensors["k_scale"].copy_(torch.from_numpy(self.k_scale))
        self.tensors["v_scale"].copy_(torch.from_numpy(self.v_scale))


def _starts(new):
    return [0] + list(np.cumsum(new))


def _check(got, want, bounds, label):
    for name, g, w, bound in zip(("out", "m", "l"), got, want, bounds):
        g = _np(g)
        rows = bound >= 0
        assert np.array_equal(np.isnan(g[rows]), np.isnan(w[rows])), f"{label}: NaN in other places of {name}"
        fine = rows & np.isfinite(w)
        assert np.array_equal(g[rows & np.isinf(w)], w[rows & np.isinf(w)]), f"{label}: infinities of {name}"
        off = np.abs(g[fine] - w[fine]) - bound[fine]
        assert not fine.any() or off.max() <= 0, f"{label}: {name} is {off.max():.3g} past its bound"


def _attend(cache, q, new, causal=True, scale=None, seq_lens=None, starts=None, label="", **kw):
    """Calls the operator and compares with the definition; returns the outputs."""
    import pmkl_amd

    seq_lens = cache.lengths if seq_lens is None else seq_lens
    starts = _starts(new) if starts is None else starts
    got = pmkl_amd.cache_attn_fwd(q, **cache.tensors, block_table=_int32(cache.table), seq_lens=_int32(seq_lens),
                                  query_start=_int32(starts), is_causal=causal, scale=scale, **kw)
    name = {"torch.float32": "fp32", "torch.float16": "fp16", "torch.bfloat16": "bf16"}[str(q.dtype)]
    real = float(np.float32(scale)) if scale else float(np.float32(1) / np.sqrt(np.float32(q.shape[2])))
    want, bounds = ref.attend(_np(q), cache.k, cache.v, cache.k_scale, cache.v_scale, cache.table, seq_lens, starts, causal,
                              real, name)
    _check(got, want, bounds, label)
    return got


def _q(tokens, heads, dim, dtype, seed):
    import torch

    x = np.random.default_rng(seed).normal(size=(tokens, heads, dim))
    return torch.from_numpy(x).to(_dtype(dtype)).to("cuda:0")


# ------------------------------------------------------------------------------------------------ attention

@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("page,kv_heads,group", [(16, 2, 4), (64, 1, 1), (256, 3, 5)])
def test_single_tokens(device, dtype, dim, page, kv_heads, group):
    """One token to a request, at every kind of end of a tile and a page; a request without tokens in the cache sees
    nothing."""
    lengths = [1, 15, 16, 17, 63, 64, 65, 127, 200, 300, 0]
    _say(f"single tokens {dtype} D{dim} page {page} heads {kv_heads}x{group}")
    cache = Cache(lengths, kv_heads, page, dim, seed=dim + page)
    q = _q(len(lengths), kv_heads * group, dim, dtype, seed=1)
    out, m, l = _attend(cache, q, [1] * len(lengths), label=f"{dtype} {dim} {page}")
    assert not out[-1].any() and (m[-1] == -math.inf).all() and not l[-1].any()


@pytest.mark.parametrize("dtype,dim,page,kv_heads,group", [
    ("bf16", 128, 16, 2, 4), ("fp16", 64, 32, 1, 20), ("fp32", 32, 128, 3, 1), ("fp32", 128, 16, 1, 7), ("bf16", 64, 64, 2, 16)])
@pytest.mark.parametrize("causal", [True, False])
def test_many_tokens(device, dtype, dim, page, kv_heads, group, causal):
    """Requests that bring none, one or many tokens, some their whole length, with more query rows than a tile holds."""
    lengths, new = [37, 130, 70, 64, 1, 260], [5, 0, 70, 1, 1, 41]
    _say(f"many tokens {dtype} D{dim} page {page} causal={causal}")
    cache = Cache(lengths, kv_heads, page, dim, seed=7, interleaved=True)
    _attend(cache, _q(sum(new), kv_heads * group, dim, dtype, seed=2), new, causal=causal, label=f"{dtype} {dim} {causal}")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_long_contexts(device, dtype):
    """Contexts of thousands of tokens beside short ones."""
    lengths, new = [5000, 3, 2049, 700], [1, 1, 1, 3]
    _say(f"long contexts {dtype}")
    cache = Cache(lengths, 2, 16, 64, seed=9)
    _attend(cache, _q(sum(new), 8, 64, dtype, seed=3), new, label=dtype)


def _form(cache, q):
    """The kernels that the library chooses for these sizes."""
    from pmkl_amd import capi

    pages, kv_heads, page, dim = cache.k.shape
    a = capi.make_cache_attn_args(capi.make_kv_cache(0, 0, 0, 0, pages=pages, kv_heads=kv_heads, page_size=page, head_dim=dim),
                                  dtype={2: capi.PMKL_DTYPE_BF16, 4: capi.PMKL_DTYPE_F32}[q.element_size()],
                                  tokens=q.shape[0], heads=q.shape[1], batch=cache.table.shape[0],
                                  table_width=cache.table.shape[1])
    names = capi.cache_attn_kernel_name(a)
    return "chunk" if "_chunk_" in names else "split" if "_split_" in names else "whole"


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dim,page,kv_heads,group,causal", [
    (128, 16, 4, 8, True), (64, 128, 8, 4, True), (32, 32, 16, 3, True), (128, 64, 2, 16, False)])
def test_chunks(device, dtype, dim, page, kv_heads, group, causal):
    """Chunks of prompts beside single tokens, in the form for calls of many rows: chunks that fill their row blocks or
    not, with and without cached tokens before them, of the whole request and longer than what is cached; a hidden page
    in one, a NaN value in another, scales far apart in a third."""
    _say(f"chunks {dtype} D{dim} page {page} heads {kv_heads}x{group} causal={causal}")
    new = [520, 1, 129, 300, 0, 64, 1, 90]
    lengths = [1100, 700, 129, 640, 50, 65, 1, 30]
    cache = Cache(lengths, kv_heads, page, dim, seed=dim + page, interleaved=page == 64)
    cache.table[0, 300 // page] = -1
    page3, off = cache.table[3, 500 // page], 500 % page
    cache.v[page3, 0, 7, off] = 0x7f
    cache.v_scale[cache.table[2, 0]] *= 2.0 ** 30 if dtype != "fp16" else 2.0 ** 4
    cache.v_scale[cache.table[5, -(-65 // page) - 1]] *= 2.0 ** -30
    cache.refresh()
    # rows of no request make it a call of many rows
    q = _q(max(sum(new) + 10, 2 ** 23 // (kv_heads * group * dim) + 1), kv_heads * group, dim, dtype, seed=dim)
    assert _form(cache, q) == "chunk"
    out, m, l = _attend(cache, q, new, causal=causal, label=f"{dtype} {dim}")
    if causal:
        # request 3: rows 650 .. 949 stand at 340 .. 639
        assert not out[650:810].isnan().any() and out[810:950, :group, 7].isnan().all()


def test_forms(device):
    """The sizes of these tests reach every form."""
    for lengths, tokens, heads, form in (([1500], 1, 4, "whole"), ([1600], 1, 4, "split"), ([300], 2100, 32, "chunk")):
        assert _form(Cache(lengths, 2, 16, 64, seed=1, width_more=0), _q(tokens, heads, 64, "bf16", 1)) == form


def test_one_long_request(device):
    lengths = [20000]
    cache = Cache(lengths, 1, 32, 128, seed=10)
    _attend(cache, _q(1, 3, 128, "bf16", seed=4), [1], label="one request")


@pytest.mark.parametrize("causal", [True, False])
def test_rows_before_the_first_token_see_nothing(device, causal):
    """More new tokens than the cache has: causal, the first of them stand before its first token."""
    lengths, new = [3, 20], [10, 20]
    cache = Cache(lengths, 2, 16, 64, seed=11)
    out, m, l = _attend(cache, _q(30, 4, 64, "bf16", seed=5), new, causal=causal, label=f"causal={causal}")
    if causal:
        assert not out[:7].any() and (m[:7] == -math.inf).all() and not l[:7].any()


@pytest.mark.parametrize("bad", [-1, -2**31, 10**6, 2**31 - 1])
def test_pages_outside_the_cache_are_hidden(device, bad):
    """Single pages, the first tokens, the last and all of them; tokens past the table's width too."""
    lengths = [200, 200, 200, 90, 200]
    cache = Cache(lengths, 2, 16, 32, seed=12)
    cache.table[0, 3], cache.table[0, 9] = bad, bad
    cache.table[1, :6] = bad
    cache.table[2, 10:] = bad
    cache.table[3, :] = bad
    cache.table = cache.table[:, :11].copy()
    out, m, l = _attend(cache, _q(5, 6, 32, "fp16", seed=6), [1] * 5, label=f"page {bad}")
    assert not out[3].any() and (l[3] == 0).all()


def test_nan_in_later_tokens_stays_there(device):
    """A NaN key or value of a new token reaches the rows that see the token, and no row before it."""
    cache = Cache([100, 90], 2, 32, 64, seed=13)
    for b, at in ((0, 90), (1, 75)):
        page, off = cache.table[b, at // 32], at % 32
        if b == 0:
            cache.v[page, 1, 5, off] = 0x7f
            cache.v[page, 0, 40, off] = 0xff
        else:
            cache.k[page, 0, off, 3] = 0x7f
    cache.refresh()
    out, m, l = _attend(cache, _q(60, 4, 64, "bf16", seed=7), [30, 30], label="NaN")
    # request 0: rows 0 .. 29 stand at 70 .. 99; request 1: rows 30 .. 59 at 60 .. 89
    assert not out[:20].isnan().any() and out[20:30, 2:, 5].isnan().all() and out[20:30, :2, 40].isnan().all()
    assert not out[30:45].isnan().any() and out[45:, :2].isnan().all() and not out[45:, 2:].isnan().any()


def test_nan_and_infinite_queries_keep_to_their_rows(device):
    cache = Cache([70, 70], 1, 16, 128, seed=14)
    q = _q(2, 4, 128, "bf16", seed=8)
    clean = [x.clone() for x in _attend(cache, q, [1, 1], label="clean")]
    q[0, 1, 7] = math.nan
    q[1, 2, 0] = math.inf
    import pmkl_amd

    got = pmkl_amd.cache_attn_fwd(q, **cache.tensors, block_table=_int32(cache.table), seq_lens=_int32([70, 70]),
                                  query_start=_int32([0, 1, 2]))
    assert got[0][0, 1].isnan().all() and got[0][1, 2].isnan().all()
    for a, b in zip(got, clean):
        for t, h in ((0, 0), (0, 2), (0, 3), (1, 0), (1, 1), (1, 3)):
            assert (a[t, h] == b[t, h]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_scales_far_apart(device, dtype):
    """Pages of one head whose scales differ by 2^80, the larger ones with and without weight."""
    cache = Cache([160], 2, 16, 64, seed=15)
    for w, e in enumerate((0, -40, 40, 0, -40, 40, 0, 0, 20, -20)):
        cache.v_scale[cache.table[0, w]] *= 2.0 ** e if dtype != "fp16" else 2.0 ** (e // 8)
        cache.k_scale[cache.table[0, w]] *= 2.0 ** (-abs(e) / 8)
    cache.refresh()
    _attend(cache, _q(4, 4, 64, dtype, seed=9), [4], scale=0.3, label=dtype)


def test_strides_and_given_buffers(device):
    """Queries from a packed projection, outputs into a view of a larger buffer; rows of no request stay as they were."""
    import torch

    lengths, new = [50, 33], [3, 2]
    cache = Cache(lengths, 2, 16, 64, seed=16, interleaved=True)
    packed = _q(9, 3 * 4, 64, "fp16", seed=10).view(9, 3, 4, 64)
    q = packed[:, 1]
    big = torch.full((9, 8, 64), 7.0, dtype=torch.float16, device="cuda:0")
    m, l = (torch.full((9, 4), 7.0, device="cuda:0") for _ in range(2))
    got = _attend(cache, q, new, starts=[0, 3, 5], out=big[:, 2:6], out_m=m, out_l=l, label="buffers")
    assert got[0].data_ptr() == big[:, 2:6].data_ptr() and got[1] is m or got[1].data_ptr() == m.data_ptr()
    assert (big[5:] == 7).all() and (big[:, :2] == 7).all() and (big[:, 6:] == 7).all() and (m[5:] == 7).all() and (l[5:] == 7).all()
    # what the kernels cannot address is copied: expanded and transposed queries
    one = _q(1, 4, 64, "fp16", seed=11)
    _attend(cache, one.expand(5, 4, 64), new, label="expanded")
    turned = _q(64, 4, 5, "fp16", seed=12).permute(2, 1, 0)
    _attend(cache, turned, new, label="turned")


def test_results_of_one_allocation(device):
    """Results that are not given lie in one allocation, apart from each other; each is an ordinary tensor that outlives
    the others, also in inference mode and without tokens."""
    import torch

    import pmkl_amd

    cache = Cache([50, 33], 2, 16, 32, seed=23)
    q = _q(5, 2, 32, "fp16", seed=23)
    given = torch.full((5, 2), 7.0, device="cuda:0")
    with torch.inference_mode():
        a = _attend(cache, q, [3, 2], out_m=given, label="inference")
    b = _attend(cache, q, [3, 2], label="all")
    assert a[1] is given or a[1].data_ptr() == given.data_ptr()
    for x, y in zip(a, b):
        assert x.is_contiguous() and y.is_contiguous() and (x == y).all()
    spans = sorted((x.data_ptr(), x.data_ptr() + x.numel() * x.element_size()) for x in b)
    assert all(e <= s for (_, e), (s, _) in zip(spans, spans[1:]))
    m = b[1]
    want = m.clone()
    b[0].add_(1), b[2].zero_()
    del b
    junk = [torch.full((4096,), 3.0, device="cuda:0") for _ in range(8)]
    assert (m == want).all() and m.requires_grad is False and len(junk) == 8
    (m.clone().requires_grad_(True) * 2).sum().backward()
    none = pmkl_amd.cache_attn_fwd(q[:0], **cache.tensors, block_table=_int32(cache.table), seq_lens=_int32([50, 33]),
                                   query_start=_int32([0, 0, 0]))
    assert [tuple(x.shape) for x in none] == [(0, 2, 32), (0, 2), (0, 2)]
    lens, start, slots, head = pmkl_amd.cache_slots(_int32([0]), _int32([0]), _int32([[-1]]), _int32([0]), _int32([5]), 16, 0)
    assert lens.tolist() == [0] and start.tolist() == [0, 0] and slots.shape == (0,) and head.tolist() == [5]
    with pytest.raises(RuntimeError, match="2\\^31"):
        pmkl_amd.cache_slots(_int32([0]), _int32([0]), _int32([[-1]]), _int32([0]), _int32([5]), 16, 2 ** 61)


def test_starts_past_the_rows_are_clamped(device):
    import torch

    cache = Cache([40, 40, 40], 1, 16, 32, seed=17)
    q = _q(4, 2, 32, "bf16", seed=13)
    out = torch.full((4, 2, 32), 7.0, dtype=q.dtype, device="cuda:0")
    import pmkl_amd

    for starts in ([0, 2, 9, 2**31 - 1], [-5, 2, 4, 4], [0, 0, 0, 0]):
        out.fill_(7.0)
        pmkl_amd.cache_attn_fwd(q, **cache.tensors, block_table=_int32(cache.table), seq_lens=_int32([40, 40, 2**31 - 1]),
                                query_start=_int32(starts), out=out)
        torch.cuda.synchronize()
        assert (out == 7).all() == (starts == [0, 0, 0, 0])


@pytest.mark.parametrize("width_more,tokens", [(0, 0), (200, 0), (0, 2200)])
def test_starts_that_fall(device, width_more, tokens):
    """query_start must not decrease.  Where it does nothing but the call's rows is written, in every form, however often
    requests name the same rows."""
    import torch

    import pmkl_amd

    cache = Cache([40] * 70, 1, 16, 64, seed=21, width_more=width_more)
    tokens = tokens or 70
    q = _q(tokens, 32, 64, "bf16", seed=21)
    big = torch.full((tokens + 2, 32, 64), 7.0, dtype=q.dtype, device="cuda:0")
    for starts in ([tokens] + [0] * 70, [0, tokens] * 35 + [0], list(range(71))[::-1], [0] * 66 + [2**31 - 1, -2**31] * 2 + [0]):
        pmkl_amd.cache_attn_fwd(q, **cache.tensors, block_table=_int32(cache.table), seq_lens=_int32([40] * 70),
                                query_start=_int32(starts), out=big[1:-1])
    torch.cuda.synchronize()
    assert (big[0] == 7).all() and (big[-1] == 7).all()


@pytest.mark.parametrize("longest", [700, 2000])
def test_many_requests(device, longest):
    """More requests than a wave has lanes, some of no tokens, their lengths far apart, in the whole and the split form."""
    rng = np.random.default_rng(22)
    lengths = [int(longest ** rng.uniform()) for _ in range(149)] + [longest]
    new = [int(rng.choice([0, 1, 1, 1, min(n, 5)])) for n in lengths]
    cache = Cache(lengths, 2, 16, 64, seed=22, width_more=0)
    q = _q(sum(new), 4, 64, "fp16", seed=22)
    assert _form(cache, q) == ("whole" if longest < 1000 else "split")
    _attend(cache, q, new, label=f"{longest}")


def test_offsets_past_32_bits(device):
    """Pages 300 MiB apart: the last ones lie past 4 GiB; and a token stride of 1 MiB within a page."""
    import torch

    page, dim = 16, 64
    small = Cache([150, 130], 1, page, dim, seed=18, spare=0)
    pages = small.k.shape[0]
    stride = 300 << 20
    store = torch.empty((pages * stride,), dtype=torch.uint8, device="cuda:0")
    k = store.as_strided((pages, 1, page, dim), (stride, 64, 1 << 20, 1))
    v = store[1 << 10:].as_strided((pages, 1, dim, page), (stride, 64, 1 << 20, 1))
    k.copy_(torch.from_numpy(small.k))
    v.copy_(torch.from_numpy(small.v))
    small.tensors["k_cache"], small.tensors["v_cache"] = (x.view(torch.float8_e4m3fn) for x in (k, v))
    _attend(small, _q(2, 4, dim, "bf16", seed=14), [1, 1], label="64-bit offsets")
    slot = np.array([small.table[0, 9] * page + 6, small.table[1, 8] * page + 2])
    x, y = _q(2, 1, dim, "bf16", seed=15), _q(2, 1, dim, "bf16", seed=16)
    import pmkl_amd

    pmkl_amd.cache_append(x, y, torch.from_numpy(slot).to("cuda:0"), **small.tensors)
    want = ref.append(_np(x), _np(y), slot, small.k, small.v, small.k_scale, small.v_scale)
    assert np.array_equal(k.cpu().numpy(), want[0]) and np.array_equal(v.cpu().numpy(), want[1])


def test_the_same_call_gives_the_same_bits(device):
    import torch

    import pmkl_amd

    lengths = [3000, 17, 900, 64] * 4
    cache = Cache(lengths, 4, 16, 128, seed=19)
    q = _q(len(lengths), 16, 128, "bf16", seed=17)
    args = dict(**cache.tensors, block_table=_int32(cache.table), seq_lens=_int32(lengths),
                query_start=_int32(_starts([1] * len(lengths))))
    first = [x.clone() for x in pmkl_amd.cache_attn_fwd(q, **args)]
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, pmkl_amd.cache_attn_fwd(q, **args)))


# ------------------------------------------------------------------------------------------------ appends

def _append_both(cache, k, v, slot, label):
    import torch

    import pmkl_amd

    want = ref.append(_np(k), _np(v), slot, cache.k, cache.v, cache.k_scale, cache.v_scale)
    pmkl_amd.cache_append(k, v, torch.from_numpy(np.asarray(slot, dtype=np.int64)).to("cuda:0"), **cache.tensors)
    names = ("k_cache", "v_cache", "k_scale", "v_scale")
    for name, w in zip(names, want):
        t = cache.tensors[name]
        if w.dtype == np.uint8:
            g = ref.E4M3[_codes(t)]
            w = ref.E4M3[w]
        else:
            g = _np(t)
        same = (g == w) | (np.isnan(g) & np.isnan(w))
        assert same.all(), f"{label}: {name} differs at {np.argwhere(~same)[:4].tolist()}"
    cache.k, cache.v, cache.k_scale, cache.v_scale = want[0], want[1], want[2].astype(np.float32), want[3].astype(np.float32)


def _slots_of(cache, page, b, first, count):
    at = np.arange(first, first + count)
    return cache.table[b, at // page] * page + at % page


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dim,page,kv_heads", [(32, 16, 3), (64, 32, 2), (128, 16, 1), (128, 256, 2), (64, 128, 1),
                                               (32, 256, 2), (128, 64, 3)])
def test_append(device, dtype, dim, page, kv_heads):
    """Runs of one token, of part of a page, over several pages, in the middle of a page whose scale has to grow or not;
    skipped slots between and around them; views of a packed projection."""
    import torch

    _say(f"append {dtype} D{dim} page {page} heads {kv_heads}")
    lengths = [2 * page + 5, page, 5 * page, 3 * page - 1, 300]
    cache = Cache(lengths, kv_heads, page, dim, seed=dim + page, interleaved=page == 32)
    pieces = [_slots_of(cache, page, 0, 2 * page + 3, 2), [-1], _slots_of(cache, page, 1, page - 1, 1),
              _slots_of(cache, page, 2, page // 2, 3 * page + 1), [cache.k.shape[0] * page, -7, 2**62],
              _slots_of(cache, page, 3, 0, 3 * page - 1), _slots_of(cache, page, 4, 290, 10)]
    slot = np.concatenate(pieces)
    rng = np.random.default_rng(20)
    x = rng.normal(size=(len(slot), 3, kv_heads, dim)) * 2.0 ** rng.integers(-6, 7, size=(len(slot), 1, 1, 1))
    packed = torch.from_numpy(x).to(_dtype(dtype)).to("cuda:0")
    _append_both(cache, packed[:, 0], packed[:, 2], slot, f"{dtype} {dim} {page}")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_append_values_at_the_borders(device, dtype):
    """Zeros, the least and the largest numbers, ties, values next to 448 times a power of two, infinities and NaN."""
    import torch

    dim, page = 32, 16
    cache = Cache([40], 1, page, dim, seed=21)
    top = float(torch.finfo(_dtype(dtype)).max)
    tiny = float(torch.finfo(_dtype(dtype)).tiny)
    rows = [np.zeros(dim), np.full(dim, tiny), np.full(dim, top), np.r_[448.0, np.linspace(1, 30, dim - 1)],
            np.r_[452.0, np.full(dim - 1, 1.0625)], np.r_[math.inf, -math.inf, math.nan, np.ones(dim - 3)],
            np.full(dim, -math.inf), np.r_[224.0, np.arange(dim - 1) + 0.5], np.r_[-3e-5, np.full(dim - 1, 7.0)]]
    for i, row in enumerate(rows):
        for at in (0, 5, 15):       # a page's first token, one of its middle, its last
            x = torch.from_numpy(np.broadcast_to(row, (1, 1, dim)).copy()).to(_dtype(dtype)).to("cuda:0")
            _append_both(cache, x, -x, _slots_of(cache, page, 0, at, 1), f"row {i} at {at}")


def test_append_forgets_a_page_that_starts_anew(device):
    """A page that an earlier request left with large values: its first token sets the scale, and one behind a scale that
    is no positive number does too."""
    import torch

    cache = Cache([32], 1, 16, 32, seed=22)
    for value, at in ((1e30, 0), (1.0, 0), (2.0, 1)):
        x = torch.full((1, 1, 32), value, device="cuda:0")
        _append_both(cache, x, x, _slots_of(cache, 16, 0, at, 1), f"{value} at {at}")
    for bad in (math.nan, math.inf, 0.0, -1.0):
        cache.k_scale[:] = cache.v_scale[:] = bad
        cache.refresh()
        x = torch.full((1, 1, 32), 3.0, device="cuda:0")
        _append_both(cache, x, x, _slots_of(cache, 16, 0, 20, 1), f"scale {bad}")


@pytest.mark.parametrize("page,batch", [(16, 700), (64, 300), (256, 4), (256, 3), (64, 1)])
def test_append_many_runs(device, page, batch):
    """More runs than a launch has waves for, in one call, and so few or many in large pages that waves share them or not."""
    import torch

    cache = Cache([page] * batch, 9, page, 32, seed=23)
    slot = np.array([cache.table[b, 0] * page + b % page for b in range(batch)])
    x = torch.from_numpy(np.random.default_rng(24).normal(size=(batch, 2, 9, 32))).to(torch.float16).to("cuda:0")
    _append_both(cache, x[:, 0], x[:, 1], slot, "runs")


# ------------------------------------------------------------------------------------------------ tables

def _slots_both(cached, new, table, free, head, page, tokens, label):
    import pmkl_amd

    device_table = _int32(table)
    got = pmkl_amd.cache_slots(_int32(cached), _int32(new), device_table, _int32(free), _int32([head]), page, tokens)
    want = ref.slots(cached, new, table, free, head, page, tokens)
    for name, g, w in zip(("seq_lens", "query_start", "slots", "free_head"), got, want):
        assert np.array_equal(g.cpu().numpy().reshape(-1), np.atleast_1d(w)), f"{label}: {name}"
    assert np.array_equal(device_table.cpu().numpy(), want[4]), f"{label}: table"
    return got


@pytest.mark.parametrize("batch", [1, 2, 63, 64, 255, 256, 257, 700])
@pytest.mark.parametrize("page,most", [(16, 1), (32, 40), (256, 700)])
def test_slots(device, batch, page, most):
    rng = np.random.default_rng(batch + page)
    cached = rng.integers(0, 300, batch)
    new = rng.integers(0, most + 1, batch)
    width = 1200 // page + 2
    held = -(-cached // page)
    order = rng.permutation(int((-(-(cached + new) // page)).sum()) + 5)
    table = np.full((batch, width), -1)
    at = 0
    for b in range(batch):
        table[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
    free = np.r_[999999, order[at:]]
    _slots_both(cached, new, table, free, 1, page, int(new.sum()), "exact")
    _slots_both(cached, new, table, free, 1, page, int(new.sum()) + 300, "padded")
    _slots_both(cached, new, table, free, 1, page, max(int(new.sum()) - 7, 0), "fewer rows")
    _slots_both(cached, new, table, free[:len(free) // 2], 1, page, int(new.sum()), "short list")
    _slots_both(cached, new, table[:, :held.max()], free, 1, page, int(new.sum()), "narrow table")


def test_slots_odd_values(device):
    """Nothing at all, an empty list, heads and lengths out of range, a long request."""
    _slots_both([], [], np.zeros((0, 4), int), [1, 2], 0, 16, 5, "no requests")
    _slots_both([0, 5], [0, 0], np.full((2, 3), -1), [], 0, 16, 0, "no tokens")
    _slots_both([3], [4], np.full((1, 1), 2), [], 7, 16, 4, "in the page it has")
    _slots_both([-5, 2], [3, -9], np.full((2, 2), -1), [4, 5], 0, 16, 3, "negative lengths")
    _slots_both([0], [40], np.full((1, 4), -1), [4, 5, 6], -1, 16, 40, "negative head")
    _slots_both([0], [40], np.full((1, 4), -1), [4, 5, 6], 2, 16, 40, "list ends")
    _slots_both([0], [20], np.full((1, 0), -1), [4, 5, 6], 0, 16, 20, "no table")
    _slots_both([10, 0], [200000, 3], np.full((2, 13000), -1), np.arange(14000)[::-1].copy(), 0, 16, 200003, "long request")


def test_slots_sums_past_32_bits(device):
    import pmkl_amd

    big = 2**31 - 1
    table = _int32(np.full((4, 3), -1))
    seq_lens, starts, slots, head = pmkl_amd.cache_slots(_int32([0, 5, 0, 1]), _int32([20, big, big, 7]), table,
                                                         _int32(np.arange(20)), _int32([0]), 16, 60)
    assert seq_lens.tolist() == [20, big, big, 8] and starts.tolist() == [0, 20, big, big, big]
    assert head.tolist() == [7] and table.tolist() == [[0, 1, -1], [-1, 2, 3], [4, 5, 6], [-1, -1, -1]]
    # request 1 has a token in a page that its row does not name: no slots up to the page's end
    assert slots[:20].tolist() == list(range(20)) and (slots[20:31] == -1).all() and slots[31:60].tolist() == list(range(32, 61))


# ------------------------------------------------------------------------------------------------ together

def _steps():
    """Lengths that a small server's four requests bring, step by step; the third is new in step 2, the second ends."""
    return [[37, 5, 0, 64], [1, 1, 0, 1], [1, 0, 50, 1], [1, 0, 1, 1], [0, 0, 1, 3]]


class Server:
    def __init__(self, page=16, kv_heads=2, group=3, dim=64, dtype="bf16", seed=30):
        import torch

        self.page, self.kv_heads, self.group, self.dim, self.dtype = page, kv_heads, group, dim, dtype
        self.cache = Cache([0, 0, 0, 0], kv_heads, page, dim, seed=seed, spare=24, width_more=9)
        self.table = _int32(self.cache.table)
        self.free = _int32(np.random.default_rng(seed).permutation(24))
        self.head, self.lens = _int32([0]), _int32([0, 0, 0, 0])
        self.torch = torch

    def inputs(self, new, seed, rows=None):
        rows = sum(new) if rows is None else rows
        return (_q(rows, self.kv_heads * self.group, self.dim, self.dtype, seed),
                _q(rows, self.kv_heads, self.dim, self.dtype, seed + 1) * 3, _q(rows, self.kv_heads, self.dim, self.dtype, seed + 2))

    def step(self, new, q, k, v):
        """A serving step as a program makes it, on device data alone."""
        import pmkl_amd

        t = self.cache.tensors
        seq_lens, starts, slots, head = pmkl_amd.cache_slots(self.lens, new, self.table, self.free, self.head, self.page,
                                                             q.shape[0])
        pmkl_amd.cache_append(k, v, slots, **t)
        out = pmkl_amd.cache_attn_fwd(q, **t, block_table=self.table, seq_lens=seq_lens, query_start=starts)
        self.lens.copy_(seq_lens)
        self.head.copy_(head)
        return out, slots, starts


@pytest.mark.parametrize("dtype,dim,page", [("bf16", 64, 16), ("fp32", 32, 32), ("fp16", 128, 16)])
def test_serving_steps(device, dtype, dim, page):
    server = Server(page=page, dim=dim, dtype=dtype)
    lens = np.zeros(4, int)
    table, head = server.cache.table, 0
    for i, new in enumerate(_steps()):
        _say(f"step {i} {dtype} D{dim}")
        q, k, v = server.inputs(new, seed=40 + 10 * i)
        (out, m, l), slots, starts = server.step(_int32(new), q, k, v)
        lens, want_starts, want_slots, head, table = ref.slots(lens, new, table, server.free.tolist(), head, page, sum(new))
        assert np.array_equal(slots.cpu().numpy(), want_slots) and np.array_equal(server.table.cpu().numpy(), table)
        c = server.cache
        c.k, c.v, ks, vs = ref.append(_np(k), _np(v), want_slots, c.k, c.v, c.k_scale, c.v_scale)
        c.k_scale, c.v_scale = ks.astype(np.float32), vs.astype(np.float32)
        want, bounds = ref.attend(_np(q), c.k, c.v, c.k_scale, c.v_scale, table, lens, want_starts, True,
                                  float(np.float32(1) / np.sqrt(np.float32(dim))), dtype)
        _check((out, m, l), want, bounds, f"step {i}")


def test_a_captured_decoding_step_replays(device):
    """A decoding step in a graph, its batch padded by two rows, replayed with other inputs between eager work: the state
    moves on with every replay, and every replay equals the same eager steps."""
    import torch

    eager, captured = Server(seed=31), Server(seed=31)
    first = [37, 5, 1, 64]
    for s in (eager, captured):
        s.step(_int32(first), *s.inputs(first, seed=50))
    new = _int32([1, 1, 0, 1])
    rows = 5
    held = [x.clone() for x in captured.inputs([1], seed=60, rows=rows)]
    saved = [x.clone() for x in (captured.lens, captured.head, captured.table, *captured.cache.tensors.values())]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        captured.step(new, *held)        # warm-up
    torch.cuda.current_stream().wait_stream(stream)
    for x, y in zip((captured.lens, captured.head, captured.table, *captured.cache.tensors.values()), saved):
        x.view(torch.uint8).copy_(y.view(torch.uint8)) if x.dtype == torch.float8_e4m3fn else x.copy_(y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results, slots, _ = captured.step(new, *held)
    for i in range(20):                  # over the ends of pages
        fresh = captured.inputs([1], seed=70 + i, rows=rows)
        for x, y in zip(held, fresh):
            x.copy_(y)
        for r in results:
            r[3:].fill_(7.0)             # rows of no request
        graph.replay()
        torch.cuda.synchronize()
        want, want_slots, _ = eager.step(new, *fresh)
        torch.cuda.synchronize()
        assert torch.equal(slots, want_slots) and (slots[3:] == -1).all()
        for a, b in zip(results, want):
            assert torch.equal(a[:3], b[:3]), f"replay {i}"
            assert (a[3:] == 7).all()
    assert torch.equal(captured.lens, eager.lens) and torch.equal(captured.table, eager.table)


def test_two_graphs_and_a_side_stream(device):
    """Two captured calls and an eager one on a stream of its own, all under way at once, do not disturb each other."""
    import torch

    import pmkl_amd

    lengths = [6000, 2500, 33]
    caches = [Cache(lengths, 2, 16, 64, seed=s) for s in (32, 33, 34)]
    qs = [_q(3, 8, 64, "bf16", seed=s) for s in (35, 36, 37)]
    args = [dict(**c.tensors, block_table=_int32(c.table), seq_lens=_int32(lengths), query_start=_int32([0, 1, 2, 3]))
            for c in caches]
    want = [[x.clone() for x in pmkl_amd.cache_attn_fwd(q, **a)] for q, a in zip(qs, args)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(pmkl_amd.cache_attn_fwd(qs[i], **args[i]))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(10):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            third = pmkl_amd.cache_attn_fwd(qs[2], **args[2])
        torch.cuda.synchronize()
        for got, w in zip((*outs, third), want):
            assert all(torch.equal(a, b) for a, b in zip(got, w))


# ------------------------------------------------------------------------------------------------ refusals

def test_torch_refusals(device):
    """What the bindings refuse by themselves, with tensors on the device (nothing is launched)."""
    import torch

    import pmkl_amd

    cache = Cache([20], 2, 16, 64, seed=38)
    t = cache.tensors
    q = _q(1, 4, 64, "bf16", seed=39)
    k = _q(1, 2, 64, "bf16", seed=40)
    slot = torch.zeros(1, dtype=torch.int64, device="cuda:0")
    table, lens, starts = _int32(cache.table), _int32([20]), _int32([0, 1])

    def attend(q=q, table=table, lens=lens, starts=starts, **kw):
        a = {**t, **{n: kw.pop(n) for n in list(kw) if n in t}}
        return pmkl_amd.cache_attn_fwd(q, **a, block_table=table, seq_lens=lens, query_start=starts, **kw)

    def append(k=k, v=k, slot=slot, **kw):
        return pmkl_amd.cache_append(k, v, slot, **{**t, **kw})

    def slots(cached=lens, new=lens, table=table, free=lens, head=lens, page=16, tokens=20):
        return pmkl_amd.cache_slots(cached, new, table, free, head, page, tokens)

    cpu = torch.zeros(1, dtype=torch.int32)
    for call, pattern in [
            (lambda: attend(q=q.double()), "float32, float16 or bfloat16"), (lambda: attend(q=q[0]), "3 dimensions"),
            (lambda: attend(q=q[:, :3]), "not a multiple"), (lambda: attend(q=q[..., :32]), "head_dim of q is 32"),
            (lambda: attend(k_cache=t["k_cache"].view(torch.uint8)), "k_cache must be"),
            (lambda: attend(v_cache=t["k_cache"]), "v_cache \\[pages"), (lambda: attend(k_scale=t["k_scale"].double()), "k_scale must"),
            (lambda: attend(k_scale=t["k_scale"][:1]), "must be \\[pages, kv_heads\\]"),
            (lambda: attend(k_scale=torch.ones(1, 1, device="cuda:0").expand_as(t["k_scale"])), "must not be expanded"),
            (lambda: attend(lens=lens.long()), "seq_lens must be Int"), (lambda: attend(starts=_int32([0])), "its end"),
            (lambda: attend(table=table.repeat(2, 1)), "a row and a start"), (lambda: attend(lens=cpu), "seq_lens is on cpu"),
            (lambda: attend(scale=-1.0), "scale must be positive"), (lambda: attend(out=q[:, :2]), "out must be"),
            (lambda: attend(table=_int32(np.zeros((3, 2))).t()[:1]), "rows of block_table"),
            (lambda: append(k=k.double(), v=k.double()), "float32, float16 or bfloat16"), (lambda: append(v=k.float()), "v must be"),
            (lambda: append(k=k[:, :1], v=k[:, :1]), "must be \\[tokens, 2, 64\\]"), (lambda: append(slot=slot.int()), "slots must be"),
            (lambda: append(slot=slot.repeat(2)), "one for each token"),
            (lambda: append(v_scale=torch.ones(1, 1, device="cuda:0").expand_as(t["v_scale"])), "must not be expanded"),
            (lambda: slots(cached=lens.long()), "cached_lens must be Int"), (lambda: slots(new=_int32([1, 2])), "one entry"),
            (lambda: slots(head=_int32([0, 0])), "one element"), (lambda: slots(page=17), "power of two"),
            (lambda: slots(tokens=-1), "must not be negative"), (lambda: slots(free=cpu), "free_pages is on cpu"),
            (lambda: slots(table=table[0]), "2 dimensions")]:
        with pytest.raises(RuntimeError, match=pattern):
            call()
    # nothing to do
    out, m, l = attend(q=q[:0], starts=_int32([0, 0]))
    assert out.shape == (0, 4, 64) and m.shape == (0, 4)
    append(k=k[:0], v=k[:0], slot=slot[:0])
