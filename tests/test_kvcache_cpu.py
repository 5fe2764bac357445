"""ztcp_b200.kvcache on a CPU-only host: the library exports what its header declares, and both layers refuse invalid
arguments before touching the GPU."""
from __future__ import annotations

import ctypes as C
import os
import re

import pytest
import torch

from ztcp_b200 import build, capi, kvcache

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "ztcp_kvcache.h")
FAKE = 0x10000  # never dereferenced: validation fails before any device access


@pytest.fixture(scope="module")
def lib():
    build.build()
    return kvcache._load()


def test_exports_every_declared_symbol(lib):
    names = re.findall(r"^\s*(?:int32_t|int64_t)\s+(ztcp_\w+)\(", open(HEADER).read(), re.M)
    assert sorted(names) == sorted(kvcache.KVCACHE_SYMBOLS)
    for n in names:
        assert hasattr(lib, n), n


def cache(**kw):
    a = dict(k_pool=FAKE, v_pool=FAKE, dtype=0, reserved=0, geom=capi.geometry(64, 8, 128, 0, False), pool_pages=10,
             block_tables=FAKE, table_stride=4, max_pages=4, kv_lens=FAKE, n_seqs=2)
    a.update(kw)
    return kvcache._Cache(*a.values())


def rows(**kw):
    a = dict(q=FAKE, token_stride=4096, head_stride=128, q_starts=FAKE, total_rows=9, num_heads=32, max_q_len=8,
             scale=0.1, causal=1)
    a.update(kw)
    return kvcache._Queries(*a.values())


geo = capi.geometry
CACHE_REFUSALS = [
    (dict(k_pool=None), {}, "k_pool must not be NULL"),
    (dict(k_pool=FAKE + 8), {}, "k_pool / v_pool must be 16-byte aligned"),
    (dict(dtype=2), {}, "k_pool must be float16 or bfloat16"),
    (dict(geom=geo(64, 8, 120, 0, False)), {}, "Invalid k_pool dimensions"),
    (dict(geom=geo(0, 8, 128, 0, False)), {}, "Invalid k_pool dimensions"),
    (dict(geom=geo(64, 8, 128, 24, False)), {}, "Invalid rope_dim"),
    (dict(geom=geo(64, 8, 592, 0, False)), {}, "head_dim beyond 576"),
    (dict(pool_pages=0), {}, "KV pool geometry too large or empty"),
    (dict(n_seqs=0), {}, "batch must hold at least one sequence"),
    (dict(kv_lens=None), {}, "block_tables and kv_lens must not be NULL"),
    (dict(max_pages=5), {}, "max_pages must be positive and at most the block tables' row length"),
    ({}, dict(q=None), "q must not be NULL"),
    ({}, dict(q=FAKE + 2), "q must be 16-byte aligned with strides of multiples of 8 elements"),
    ({}, dict(token_stride=4100), "q must be 16-byte aligned with strides of multiples of 8 elements"),
    ({}, dict(total_rows=0), "queries must hold at least one row"),
    ({}, dict(q_starts=None), "without q_starts there is one row per sequence"),
    ({}, dict(num_heads=12), "query heads must be a multiple of the KV heads"),
    ({}, dict(max_q_len=0), "max_q_len must be positive"),
    ({}, dict(max_q_len=1 << 60), "max_q_len must be below 2^31"),
    ({}, dict(scale=0.0), "scale must be positive and finite"),
    ({}, dict(scale=float("nan")), "scale must be positive and finite"),
    ({}, dict(scale=float("inf")), "scale must be positive and finite"),
]


@pytest.mark.parametrize("ckw,qkw,msg", CACHE_REFUSALS)
def test_attend_and_mass_refusals(lib, ckw, qkw, msg):
    c, q = cache(**ckw), rows(**qkw)
    assert lib.ztcp_attend_workspace_bytes(c, q) == -1 and lib.ztcp_last_error().decode() == msg
    assert lib.ztcp_attend_pages(c, q, FAKE, None, FAKE, FAKE, 1 << 40, None) == capi.ZTCP_EINVAL
    assert lib.ztcp_last_error().decode() == msg
    assert lib.ztcp_page_mass(c, q, FAKE, None, 1.0, FAKE, FAKE, FAKE, 1 << 40, None) == capi.ZTCP_EINVAL
    assert lib.ztcp_last_error().decode() == msg


def test_scale_too_large_for_base_2(lib):
    """Scores enter exp2: a scale that is finite but not times log2(e) would make every score infinite."""
    c, q = cache(), rows(scale=3e38)
    msg = "scale must be positive and finite, times log2(e) too"
    assert lib.ztcp_attend_pages(c, q, FAKE, None, FAKE, FAKE, 1 << 40, None) == capi.ZTCP_EINVAL
    assert lib.ztcp_last_error().decode() == msg
    assert lib.ztcp_page_mass(c, q, FAKE, None, 1.0, FAKE, FAKE, FAKE, 1 << 40, None) == capi.ZTCP_EINVAL
    assert lib.ztcp_last_error().decode() == msg


def test_too_many_sequences(lib):
    """Beyond 2^21 sequences a kernel's start comes near the bound of its waits."""
    for n, msg in (((1 << 21) + 1, "more than 2^21 sequences in a batch"), (1 << 24, "more than 2^21 sequences in a batch"),
                   (-1, "batch must hold at least one sequence")):
        c, q = cache(n_seqs=n), rows()
        assert lib.ztcp_attend_pages(c, q, FAKE, None, FAKE, FAKE, 1 << 40, None) == capi.ZTCP_EINVAL
        assert lib.ztcp_last_error().decode() == msg
        assert lib.ztcp_page_mass(c, q, FAKE, None, 1.0, FAKE, FAKE, FAKE, 1 << 40, None) == capi.ZTCP_EINVAL
        assert lib.ztcp_last_error().decode() == msg


def test_wait_limit(lib):
    default = 2_000_000_000
    assert lib.ztcp_wait_limit(500) == default
    assert lib.ztcp_wait_limit(0) == 500
    assert lib.ztcp_wait_limit(-1) == default and lib.ztcp_wait_limit(0) == default


def test_attend_refusals(lib):
    def refuse(msg, c=None, out=FAKE, status=FAKE, ws=FAKE):
        rc = lib.ztcp_attend_pages(c or cache(), rows(), out, None, status, ws, 1 << 40, None)
        assert rc == capi.ZTCP_EINVAL and lib.ztcp_last_error().decode() == msg

    refuse("out, status and workspace must not be NULL", out=None)
    refuse("out, status and workspace must not be NULL", status=None)
    refuse("out, status and workspace must not be NULL", ws=None)
    refuse("out and workspace must be 16-byte aligned", out=FAKE + 4)
    refuse("a single-buffer pool needs rope_dim < head_dim", cache(v_pool=None, geom=geo(64, 8, 128, 128, True)))
    wide = "head_dim beyond 256 (single-buffer pools: 576, with 512 value columns)"
    refuse(wide, cache(geom=geo(64, 8, 272, 0, False)))
    refuse(wide, cache(v_pool=None, geom=geo(64, 8, 576, 0, True)))
    assert lib.ztcp_attend_pages(None, rows(), FAKE, None, FAKE, FAKE, 1, None) == capi.ZTCP_EINVAL


def test_mass_refusals(lib):
    def refuse(msg, lse=FAKE, decay=1.0, out=FAKE, status=FAKE, ws=FAKE):
        rc = lib.ztcp_page_mass(cache(), rows(), lse, None, decay, out, status, ws, 1 << 40, None)
        assert rc == capi.ZTCP_EINVAL and lib.ztcp_last_error().decode() == msg

    refuse("lse, out_mass, status and workspace must not be NULL", lse=None)
    refuse("lse, out_mass, status and workspace must not be NULL", out=None)
    refuse("lse, out_mass, status and workspace must not be NULL", ws=None)
    refuse("workspace must be 16-byte aligned", ws=FAKE + 8)
    refuse("decay must be finite", decay=float("inf"))


@pytest.mark.parametrize("kw,msg", [
    (dict(k=None), "k must not be NULL"),
    (dict(v=None), "v must be given exactly when v_pool is"),
    (dict(q_out=None), "q needs q_out and a positive number of heads"),
    (dict(k_token_stride=12), "q, k, v and q_out must be 16-byte aligned with strides of multiples of 8 elements"),
    (dict(slots=None), "slots must not be NULL"),
    (dict(rope_table=None), "a rotation needs positions and a rope table"),
    (dict(positions=None), "a rotation needs positions and a rope table"),
    (dict(q_weight=FAKE + 4), "rope_table, q_weight and k_weight must be 16-byte aligned"),
    (dict(rope_table=FAKE + 8), "rope_table, q_weight and k_weight must be 16-byte aligned"),
    (dict(norm_from=8), "norm_from must be a multiple of 16 below head_dim"),
    (dict(norm_from=128), "norm_from must be a multiple of 16 below head_dim"),
    (dict(eps=-1.0), "eps must be non-negative and finite"),
    (dict(n_tokens=0), "append must hold at least one token"),
    (dict(geom=geo(64, 8, 1040, 0, False)), "head_dim beyond 1024"),
    (dict(geom=geo(64, 8, 512, 272, False)), "rope_dim beyond 256"),
])
def test_append_refusals(lib, kw, msg):
    a = dict(q=FAKE, k=FAKE, v=FAKE, q_token_stride=4096, q_head_stride=128, k_token_stride=1024, k_head_stride=128,
             v_token_stride=1024, v_head_stride=128, q_out=FAKE, k_pool=FAKE, v_pool=FAKE, slots=FAKE, positions=FAKE,
             rope_table=FAKE, q_weight=FAKE, k_weight=FAKE, n_tokens=3, num_q_heads=32, pool_pages=4, max_pos=100,
             geom=geo(64, 8, 128, 64, False), dtype=0, norm_from=0, interleaved=0, eps=1e-6)
    a.update(kw)
    assert lib.ztcp_append_tokens(kvcache._Append(*a.values()), FAKE, None) == capi.ZTCP_EINVAL
    assert lib.ztcp_last_error().decode() == msg


@pytest.mark.parametrize("kw,msg", [
    (dict(mass=None), "mass, block_tables and kv_lens must not be NULL"),
    (dict(kept_lens=None), "selection outputs must not be NULL"),
    (dict(n_seqs=1 << 20, max_pages=1 << 12),
     "selection must hold at least one sequence and page, and fewer than 2^31 pages in all"),
    (dict(page_tokens=0), "selection must hold at least one sequence and page, and fewer than 2^31 pages in all"),
    (dict(n_seqs=1, max_pages=(1 << 31) - 1), "max_pages beyond 2^31 - 4096"),
    (dict(n_seqs=1, max_pages=(1 << 31) - 4095), "max_pages beyond 2^31 - 4096"),
    (dict(recent=0), "keep and sink must be non-negative and recent positive"),
    (dict(keep=-1), "keep and sink must be non-negative and recent positive"),
])
def test_select_refusals(lib, kw, msg):
    a = dict(mass=FAKE, block_tables=FAKE, kv_lens=FAKE, n_seqs=2, max_pages=4, page_tokens=64, keep=2, sink=1, recent=1,
             cold_blocks=FAKE, cold_index=FAKE, cold_starts=FAKE, kept_tables=FAKE, kept_mass=FAKE, kept_lens=FAKE,
             status=FAKE)
    a.update(kw)
    assert lib.ztcp_select_cold_pages(kvcache._Selection(*a.values()), None) == capi.ZTCP_EINVAL
    assert lib.ztcp_last_error().decode() == msg


def test_host_tensors_are_refused():
    k = torch.zeros((4, 16, 2, 64), dtype=torch.float16)
    q = torch.zeros((1, 4, 64), dtype=torch.float16)
    ints = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="k_pool must be a CUDA tensor"):
        kvcache.prepare_attend(q, k, k, ints[None], ints, q)
    with pytest.raises(RuntimeError, match="k_pool must be a CUDA tensor"):
        kvcache.append_tokens(q, k[0, :1], k[0, :1], k, k, ints.long(), ints, None, q)
    with pytest.raises(RuntimeError, match="mass must be a CUDA tensor"):
        kvcache.select_cold_pages(torch.zeros((1, 1)), ints[None], ints, page_tokens=16, keep=1)


def test_overlap_spans_strided_tensors():
    base = torch.zeros((8, 64))
    assert kvcache._overlap(base[:, :8], base[3:4, 4:6]) and kvcache._overlap(base[:, :8], base[:, 8:])
    assert not kvcache._overlap(base[:4], base[4:]) and not kvcache._overlap(None, base)


def test_rope_table_far_positions():
    """Entry (p, i) is cos / sin of p * base^(-2i/R) with the angle in 64 bits, rounded once."""
    t = kvcache.rope_table(70001, 32, 10000.0, device="cpu")
    p = 70000
    for i in (0, 3, 15):
        a = torch.tensor(p, dtype=torch.float64) * 10000.0 ** (-2.0 * i / 32)
        # the angle is off by a few 64-bit steps of 7e4 at most; the rest is one rounding to 32 bits
        assert abs(float(t[p, i]) - float(a.cos())) <= 2.0 ** -25 + 1e-10
        assert abs(float(t[p, 16 + i]) - float(a.sin())) <= 2.0 ** -25 + 1e-10
