"""Operators of ztcp_b200.kvcache on the GPU against plain 64-bit forms, at the sizes and masks where they can go
wrong: pages that end inside a tile, odd page sizes, rows that see nothing, empty sequences, stale NaN in unused page
rows, table entries outside the pool, strided queries, streams, graphs and prepared calls."""
from __future__ import annotations

import pytest
import torch

import kvcache_reference as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F16, BF16 = torch.float16, torch.bfloat16
ids = lambda x: str(x).replace("torch.", "").replace(" ", "")  # noqa: E731


def cpu(t):
    return None if t is None else t.cpu()


def queries(rows, heads, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((rows, heads, D), generator=g).to(dtype).to(DEV)


def run_attend(q, k, v, tables, lens, q_lens, *, scale=None, causal=True, rope_dim=0, decode=False, **kw):
    from ztcp_b200 import kvcache

    dv = k.shape[3] - (rope_dim if v is None else 0)
    out = torch.full((q.shape[0], q.shape[1], dv), 7.0, dtype=q.dtype, device=DEV)
    lse = torch.full(q.shape[:2], 7.0, dtype=torch.float32, device=DEV)
    starts = None if decode else ref.starts_of(q_lens)
    status = kvcache.attend_pages(q, k, v, tables, lens, out, lse=lse, q_starts=starts, max_q_len=max(max(q_lens), 1),
                                  rope_dim=rope_dim, scale=scale, causal=causal, **kw)
    torch.cuda.synchronize()
    return out, lse, status


def check_attend(kv, q_lens, T, H, G, D, dtype, *, mla_rope=None, causal=True, decode=False, seed=1, scale=None):
    mla = mla_rope is not None
    k, v, tables, lens = ref.make_cache(kv, T, H, D, dtype, seed, mla)
    q = queries(sum(q_lens), H * G, D, dtype, seed + 1)
    out, lse, status = run_attend(q, k, v, tables, lens, q_lens, causal=causal, rope_dim=mla_rope or 0, decode=decode,
                                  scale=scale)
    want, wl, tol, ltol = ref.attend(cpu(q), cpu(k), cpu(v), cpu(tables), kv, q_lens, D ** -0.5 if scale is None else scale,
                                     causal, mla_rope or 0)
    assert not status.any()
    ref.assert_close(lse, wl, ltol, "lse")
    ref.assert_close(out, want, tol, "out")


# ---- attention --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16], ids=ids)
@pytest.mark.parametrize("H,G,D", [(8, 4, 128), (2, 1, 64), (1, 16, 128), (3, 5, 80), (2, 2, 16), (1, 3, 256), (2, 4, 176)])
def test_decode(dtype, H, G, D):
    kv = [1, 64, 65, 0, 200, 127, 333]
    check_attend(kv, [1] * len(kv), 64, H, G, D, dtype, decode=True)


@pytest.mark.parametrize("T", [1, 5, 16, 48, 64, 100, 256])
def test_decode_page_sizes(T):
    kv = [300, 1, T, T + 1, 2 * T - 1]
    check_attend(kv, [1] * len(kv), T, 2, 4, 64, BF16, decode=True)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=ids)
@pytest.mark.parametrize("heads,D,rope", [(16, 576, 64), (5, 96, 32), (40, 576, 64), (8, 320, 0), (4, 272, 16)])
def test_single_buffer(dtype, heads, D, rope):
    kv = [1, 70, 0, 257]
    check_attend(kv, [1] * len(kv), 64, 1, heads, D, dtype, mla_rope=rope, decode=True)
    check_attend([90, 33], [7, 2], 16, 1, heads, D, dtype, mla_rope=rope)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=ids)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D,T", [(128, 64), (64, 16), (128, 128), (96, 32), (128, 8), (64, 256), (112, 24), (48, 64)])
def test_chunk(dtype, causal, D, T):
    kv, q_lens = [200, 5, 0, 130, 64, 385], [50, 5, 0, 129, 1, 3]
    check_attend(kv, q_lens, T, 2, 4, D, dtype, causal=causal)


@pytest.mark.parametrize("H,G", [(1, 1), (8, 1), (1, 8), (4, 3), (1, 32), (2, 7)])
def test_chunk_head_layouts(H, G):
    check_attend([300, 77, 140], [40, 77, 9], 64, H, G, 128, BF16)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=ids)
@pytest.mark.parametrize("D,H,G,T,causal", [(256, 2, 4, 64, True), (176, 1, 8, 16, True), (144, 2, 3, 128, False), (208, 1, 1, 40, True),
                                            (256, 1, 32, 5, True)])
def test_chunk_wide_heads(D, H, G, T, causal, dtype):
    """Chunks at head dims that have no chunk kernel: many row blocks of 16 an item's worth each."""
    check_attend([200, 5, 0, 130, 64, 385], [50, 5, 0, 129, 1, 33], T, H, G, D, dtype, causal=causal)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=ids)
@pytest.mark.parametrize("heads,D,rope,T", [(16, 576, 64, 64), (40, 576, 64, 16), (4, 96, 64, 64), (12, 320, 64, 32), (7, 128, 64, 8),
                                            (3, 192, 16, 64), (5, 576, 64, 24)])
def test_single_buffer_chunks(heads, D, rope, T, dtype):
    """Chunks over latent pages, of more rows than an item holds, at widths from one value group to eight."""
    check_attend([150, 3, 0, 70], [60, 3, 0, 21], T, 1, heads, D, dtype, mla_rope=rope)
    check_attend([33, 257], [1, 1], T, 1, heads, D, dtype, mla_rope=rope, decode=True)


def test_rows_that_see_nothing():
    # more query rows than tokens: the first rows see nothing; sequences without tokens or without rows between
    check_attend([3, 0, 10, 0, 70], [8, 4, 0, 0, 200], 64, 2, 4, 128, BF16)
    check_attend([3, 0, 10], [8, 4, 0], 64, 2, 4, 128, F16, causal=False)


@pytest.mark.parametrize("seed", range(6))
def test_random_batches(seed):
    kv, q_lens = ref.ragged(seed, 9, 700, 1 if seed % 3 == 0 else 60)
    q_lens[0] = max(q_lens[0], 1)
    check_attend(kv, q_lens, [64, 16, 32][seed % 3], [8, 2, 1][seed % 3], [4, 8, 6][seed % 3], [128, 64][seed % 2],
                 [F16, BF16][seed // 3], seed=seed)


def test_long_context_splits():
    check_attend([9000], [1], 64, 1, 2, 64, F16, decode=True)
    check_attend([6000, 4500], [33, 2], 64, 1, 4, 128, BF16)
    check_attend([5000], [1], 64, 1, 16, 576, BF16, mla_rope=64, decode=True)


@pytest.mark.parametrize("H,G,D,T,mla_rope,q_max", [
    (8, 4, 128, 64, None, 1), (8, 1, 64, 16, None, 1), (4, 8, 256, 64, None, 1), (1, 16, 576, 64, 64, 1),
    (1, 40, 576, 16, 64, 2), (8, 4, 128, 64, None, 90), (4, 8, 64, 16, None, 33), (2, 2, 128, 48, None, 9)])
def test_many_tiles_per_cta(H, G, D, T, mla_rope, q_max):
    """Batches whose every CTA passes many tiles of several items through its rings, run three times over."""
    batch = 40 if q_max == 1 else 8
    kv, q_lens = ref.ragged(D + T, batch, 5000, q_max)
    kv = [n + 1500 for n in kv]
    q_lens = [max(1, m) for m in q_lens]
    k, v, tables, lens = ref.make_large_cache(kv, T, H, D, BF16, 7, mla_rope is not None)
    q = queries(sum(q_lens), H * G, D, BF16, 8)
    out, lse, status = run_attend(q, k, v, tables, lens, q_lens, rope_dim=mla_rope or 0)
    assert not status.any()
    for _ in range(2):
        again = run_attend(q, k, v, tables, lens, q_lens, rope_dim=mla_rope or 0)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    want, wl, tol, ltol = ref.attend_large(q, k, v, tables, kv, q_lens, D ** -0.5, mla_rope or 0)
    ref.assert_close(lse, wl, ltol, "lse")
    ref.assert_close(out, want, tol, "out")


def test_large_scores():
    # a scale of 1 on 128 columns: scores of tens, one weight near 1
    check_attend([500, 260], [3, 100], 64, 2, 4, 128, BF16, scale=1.0)


@pytest.mark.parametrize("G,D,T", [(8, 128, 64), (3, 64, 16), (1, 128, 128)])
def test_many_short_items(G, D, T):
    """Items of a tile or two, of one and of two row tiles, many to a CTA: the next ones' tiles follow without a gap."""
    kv, q_lens = ref.ragged(D + T, 400, 130, 60)
    check_attend(kv, q_lens, T, 2, G, D, BF16)


@pytest.mark.parametrize("q_len", [1, 40])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=ids)
def test_growing_scores(dtype, q_len):
    """Every tile's scores lie far above the last's, so that each replaces the maximum, the last one's too."""
    kv = [700, 65]
    k, v, tables, lens = ref.make_cache(kv, 64, 1, 128, dtype, 5)
    for b, n in enumerate(kv):
        for j in range(n):
            k[tables[b, j // 64], j % 64] = k[tables[b, j // 64], j % 64] * 0.125 + 6 * j / 700
    q = queries(2 * q_len, 4, 128, dtype, 6) * 0.125 + 1
    out, lse, status = run_attend(q, k, v, tables, lens, [q_len] * 2)
    want, wl, tol, ltol = ref.attend(cpu(q), cpu(k), cpu(v), cpu(tables), kv, [q_len] * 2, 128 ** -0.5)
    assert not status.any()
    ref.assert_close(lse, wl, ltol, "lse")
    ref.assert_close(out, want, tol, "out")


@pytest.mark.parametrize("q_len", [1, 40])
def test_broadcast_queries(q_len):
    """Queries expanded over rows or heads (strides of 0) read as their copies do."""
    from ztcp_b200 import kvcache

    k, v, tables, lens = ref.make_cache([200, 77], 64, 2, 128, BF16, 5)
    one = queries(1, 8, 128, BF16, 6)
    for q in (one.expand(2 * q_len, 8, 128), one[:, :1].expand(1, 8, 128).expand(2 * q_len, 8, 128)):
        got = run_attend(q, k, v, tables, lens, [q_len] * 2)
        want = run_attend(q.contiguous(), k, v, tables, lens, [q_len] * 2)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        a, b = (torch.empty(tables.shape, device=DEV) for _ in range(2))
        for x, mass in ((q, a), (q.contiguous(), b)):
            kvcache.page_mass(x, k, tables, lens, want[1], None, mass, q_starts=ref.starts_of([q_len] * 2), max_q_len=q_len)
        assert torch.equal(a, b)


@pytest.mark.parametrize("hint", [1, 4, 16, 1000])
def test_any_length_is_computed(hint):
    """max_q_len chooses the kernel; rows beyond it, and fewer, come out right with every kernel."""
    from ztcp_b200 import kvcache

    kv, q_lens = [300, 70, 0, 513], [90, 1, 0, 17]
    k, v, tables, lens = ref.make_cache(kv, 64, 2, 128, BF16, 5)
    q = queries(sum(q_lens), 8, 128, BF16, 6)
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=DEV)
    mass = torch.empty(tables.shape, device=DEV)
    kvcache.attend_pages(q, k, v, tables, lens, out, lse=lse, q_starts=ref.starts_of(q_lens), max_q_len=hint)
    kvcache.page_mass(q, k, tables, lens, lse, None, mass, q_starts=ref.starts_of(q_lens), max_q_len=hint)
    torch.cuda.synchronize()
    want, wl, tol, ltol = ref.attend(cpu(q), cpu(k), cpu(v), cpu(tables), kv, q_lens, 128 ** -0.5, True)
    ref.assert_close(lse, wl, ltol, "lse")
    ref.assert_close(out, want, tol, "out")
    want, tol = ref.mass(cpu(q), cpu(k), cpu(tables), kv, q_lens, cpu(lse), None, 1.0, 128 ** -0.5, True)
    ref.assert_close(mass, want, tol, "mass")


def test_rows_behind_the_last_sequence_stay():
    from ztcp_b200 import kvcache

    k, v, tables, lens = ref.make_cache([100, 40], 64, 2, 128, BF16)
    q = queries(60, 8, 128, BF16, 3)
    out = torch.full((60, 8, 128), 5.0, dtype=BF16, device=DEV)
    lse = torch.full((60, 8), 5.0, device=DEV)
    kvcache.attend_pages(q, k, v, tables, lens, out, lse=lse, q_starts=ref.starts_of([30, 20]), max_q_len=30)
    torch.cuda.synchronize()
    assert bool((out[50:] == 5).all()) and bool((lse[50:] == 5).all())
    assert bool((out[:50] != 5).any()) and not bool((lse[:50] == 5).any())


@pytest.mark.parametrize("q_len", [1, 40])
def test_bad_blocks_count_as_masked(q_len):
    from ztcp_b200 import kvcache

    kv, q_lens = [200, 130, 64], [q_len] * 3
    k, v, tables, lens = ref.make_cache(kv, 64, 2, 128, BF16, 5)
    tables[0, 1] = -1
    tables[1, 0] = k.shape[0]
    q = queries(sum(q_lens), 8, 128, BF16, 6)
    with pytest.raises(RuntimeError, match="block_tables entries must lie"):
        run_attend(q, k, v, tables, lens, q_lens)
    out, lse, status = run_attend(q, k, v, tables, lens, q_lens, check_block_table=False)
    want, wl, tol, ltol = ref.attend(cpu(q), cpu(k), cpu(v), cpu(tables), kv, q_lens, 128 ** -0.5)
    assert status.tolist() == [kvcache.SEQ_BAD_BLOCK, kvcache.SEQ_BAD_BLOCK, kvcache.SEQ_OK]
    ref.assert_close(lse, wl, ltol, "lse")
    ref.assert_close(out, want, tol, "out")


def test_bad_lengths_are_clamped():
    from ztcp_b200 import kvcache

    k, v, tables, lens = ref.make_cache([128, 128, 128], 64, 2, 64, F16, 5)
    q = queries(3, 4, 64, F16, 6)
    lens.copy_(torch.tensor([-5, 1 << 30, 100], dtype=torch.int32))
    with pytest.raises(RuntimeError, match="kv_lens entries must lie"):
        run_attend(q, k, v, tables, lens, [1] * 3)
    out, lse, status = run_attend(q, k, v, tables, lens, [1] * 3, check_block_table=False)
    want, wl, tol, ltol = ref.attend(cpu(q), cpu(k), cpu(v), cpu(tables), [0, 128, 100], [1] * 3, 64 ** -0.5)
    assert status.tolist() == [kvcache.SEQ_BAD_LENGTH, kvcache.SEQ_BAD_LENGTH, kvcache.SEQ_OK]
    ref.assert_close(lse, wl, ltol, "lse")
    ref.assert_close(out, want, tol, "out")
    # starts that run backwards or past the rows
    starts = torch.tensor([0, 2, 1, 9], dtype=torch.int32, device=DEV)
    lens.fill_(100)
    status = kvcache.attend_pages(q, k, v, tables, lens, out, q_starts=starts, max_q_len=3)
    torch.cuda.synchronize()
    assert status.tolist() == [kvcache.SEQ_OK, kvcache.SEQ_BAD_LENGTH, kvcache.SEQ_BAD_LENGTH]


@pytest.mark.parametrize("q_lens", [[1, 1, 1], [50, 3, 20]])
def test_strided_queries(q_lens):
    kv = [100, 65, 300]
    k, v, tables, lens = ref.make_cache(kv, 64, 2, 128, BF16, 8)
    fused = queries(sum(q_lens), 8 + 2 + 2, 128, BF16, 9)  # one projection: query heads, then key and value heads
    q = fused[:, :8]
    out, lse, _ = run_attend(q, k, v, tables, lens, q_lens)
    out2, lse2, _ = run_attend(q.contiguous(), k, v, tables, lens, q_lens)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("q_lens", [[1] * 4, [70, 1, 33, 8]])
def test_prepared_call_streams_and_graph(q_lens):
    """A prepared call reads its tensors at every call, on any stream and from a graph, and repeats bit for bit."""
    from ztcp_b200 import kvcache

    kv = [700, 65, 300, 9]
    k, v, tables, lens = ref.make_cache(kv, 64, 2, 128, BF16, 8, poison=False)
    q = queries(sum(q_lens), 8, 128, BF16, 9)
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=DEV)
    call = kvcache.prepare_attend(q, k, v, tables, lens, out, lse=lse, q_starts=ref.starts_of(q_lens), max_q_len=70)
    call()
    torch.cuda.synchronize()
    first = out.clone()
    side = torch.cuda.Stream(DEV)
    out.zero_()
    side.wait_stream(torch.cuda.current_stream())
    call(side)
    side.synchronize()
    assert torch.equal(out, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    kv2 = [130, 64, 1, 9]
    lens.copy_(torch.tensor(kv2, dtype=torch.int32))
    q.copy_(queries(sum(q_lens), 8, 128, BF16, 10))
    graph.replay()
    torch.cuda.synchronize()
    want, wl, tol, ltol = ref.attend(cpu(q), cpu(k), cpu(v), cpu(tables), kv2, q_lens, 128 ** -0.5)
    ref.assert_close(lse, wl, ltol, "lse")
    ref.assert_close(out, want, tol, "out")


def test_calls_side_by_side():
    """Different operators, each with its own workspace, on four streams at once, as a batch of requests runs them."""
    from ztcp_b200 import kvcache

    k, v, tables, lens = ref.make_cache([900, 70, 300, 1500], 64, 2, 128, BF16, 5)
    one, chunk = queries(4, 8, 128, BF16, 6), queries(4 * 50, 8, 128, BF16, 7)
    starts = ref.starts_of([50] * 4)
    o1, o2 = torch.empty_like(one), torch.empty_like(chunk)
    l1, l2 = (torch.empty(q.shape[:2], device=DEV) for q in (one, chunk))
    kvcache.attend_pages(one, k, v, tables, lens, o1, lse=l1)
    kvcache.attend_pages(chunk, k, v, tables, lens, o2, lse=l2, q_starts=starts, max_q_len=50)
    m1, m2 = (torch.empty(tables.shape, device=DEV) for _ in range(2))
    calls = [kvcache.prepare_attend(one, k, v, tables, lens, o1, lse=torch.empty_like(l1)),
             kvcache.prepare_attend(chunk, k, v, tables, lens, o2, lse=torch.empty_like(l2), q_starts=starts, max_q_len=50),
             kvcache.prepare_page_mass(one, k, tables, lens, l1, None, m1),
             kvcache.prepare_page_mass(chunk, k, tables, lens, l2, None, m2, q_starts=starts, max_q_len=50)]
    for c in calls:
        c()
    torch.cuda.synchronize()
    want = [t.clone() for t in (o1, o2, m1, m2)]
    streams = [torch.cuda.Stream() for _ in calls]
    for t in (o1, o2, m1, m2):
        t.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s in zip(calls, streams):
            assert not c(s) is None
    torch.cuda.synchronize()
    for got, w in zip((o1, o2, m1, m2), want):
        assert torch.equal(got, w)


def test_one_shot_calls_on_another_stream():
    kv = [400, 65]
    k, v, tables, lens = ref.make_cache(kv, 64, 2, 128, BF16, 8)
    q = queries(2, 8, 128, BF16, 9)
    want, _, _ = run_attend(q, k, v, tables, lens, [1, 1])
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    for stream in (side, side.cuda_stream):
        out, _, _ = run_attend(q, k, v, tables, lens, [1, 1], stream=stream)
        assert torch.equal(out, want)


def long_work(stream=None):
    """About a tenth of a second of work on a stream (default: the current one)."""
    with torch.cuda.stream(stream):
        torch.cuda._sleep(200_000_000)


def left_over(sizes):
    """Memory that the current stream's allocator hands out next, in these sizes, and that the stream overwrites with
    ones only after its long work."""
    torch.cuda.synchronize()
    blocks = [torch.empty(n, dtype=torch.uint8, device=DEV) for n in sizes for _ in range(3)]
    long_work()
    for x in blocks:
        x.fill_(255)


@pytest.mark.parametrize("op", ["attend", "mass", "append", "select"])
def test_own_buffers_while_the_current_stream_is_busy(op):
    """A one-shot call on another stream does not take memory that the current stream's earlier work still writes; nor
    does a prepared call that runs on one."""
    from ztcp_b200 import kvcache

    kv = [1500, 65, 900]
    k, v, tables, lens = ref.make_cache(kv, 64, 2, 128, BF16, 8)
    q = queries(3 * 30, 8, 128, BF16, 9)
    starts = ref.starts_of([30] * 3)
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=DEV)
    kvcache.attend_pages(q, k, v, tables, lens, out, lse=lse, q_starts=starts, max_q_len=30)
    mass = torch.rand(tables.shape, device=DEV)
    summed = torch.empty_like(mass)
    new = queries(8000, 2 + 2, 128, BF16, 10)
    kp, vp = (torch.zeros((8000 // 64 + 1, 64, 2, 128), dtype=BF16, device=DEV) for _ in range(2))
    slots = torch.arange(8000, device=DEV)
    kw = dict(q_starts=starts, max_q_len=30, check_block_table=False)
    if op == "attend":
        args, once, prepare = (q, k, v, tables, lens, out), kvcache.attend_pages, kvcache.prepare_attend
        kw["lse"] = lse
        results = [out, lse]
    elif op == "mass":
        args, once, prepare = (q, k, tables, lens, lse.clone(), None, summed), kvcache.page_mass, kvcache.prepare_page_mass
        results = [summed]
    elif op == "append":
        args, kw = (None, new[:, :2], new[:, 2:], kp, vp, slots, None, None, None), {}
        once, prepare = kvcache.append_tokens, kvcache.prepare_append
        results = [kp, vp]
    else:
        args, kw = (mass, tables, lens), dict(page_tokens=64, keep=4)
        once, results = kvcache.select_cold_pages, []
    first = once(*args, **kw)
    torch.cuda.synchronize()
    results += list(first) if op == "select" else [first]
    want = [t.clone() for t in results]
    sizes = [t.numel() * t.element_size() for t in results]
    if op != "select":
        sizes += [t.numel() * t.element_size() for t in prepare(*args, **kw)._own]
    del first
    results = results[:len(results) if op == "select" else -1]
    side = torch.cuda.Stream(DEV)
    for prepared in (False, True):
        if prepared and op == "select":
            continue
        for t in results:
            t.zero_()
        left_over(sizes)
        got = prepare(*args, **kw)(side) if prepared else once(*args, stream=side, **kw)
        if not prepared:
            assert not torch.cuda.current_stream().query()  # the call did not wait for the current stream
        torch.cuda.synchronize()
        got = list(got) if op == "select" else [*results, got]
        for g, w in zip(got, want):
            assert torch.equal(g, w)


def test_prepared_call_dropped_while_it_runs():
    """The buffers of a prepared call that another stream still runs are not handed out."""
    from ztcp_b200 import kvcache

    kv = [1500, 65, 900]
    k, v, tables, lens = ref.make_cache(kv, 64, 2, 128, BF16, 8)
    q = queries(3, 8, 128, BF16, 9)
    out, want = torch.empty_like(q), torch.empty_like(q)
    kvcache.attend_pages(q, k, v, tables, lens, want)
    call = kvcache.prepare_attend(q, k, v, tables, lens, out)
    size = call._own[0].numel()
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    long_work(side)
    status = call(side)
    taken = call._own[0].data_ptr()
    del call
    fresh = [torch.full((size,), 255, dtype=torch.uint8, device=DEV) for _ in range(4)]
    assert taken not in [t.data_ptr() for t in fresh]
    torch.cuda.synchronize()
    assert torch.equal(out, want) and not status.any()


def test_host_check_reads_in_the_calls_stream():
    """Lengths and tables that the call's own stream has just been told to write are checked as they will be."""
    from ztcp_b200 import kvcache

    kv = [700, 65, 900]
    k, v, tables, lens = ref.make_cache(kv, 64, 2, 128, BF16, 8)
    q = queries(3, 8, 128, BF16, 9)
    want, out = torch.empty_like(q), torch.empty_like(q)
    kvcache.attend_pages(q, k, v, tables, lens, want)
    side = torch.cuda.Stream(DEV)
    late_tables, late_lens = torch.full_like(tables, -1), torch.full_like(lens, 1 << 30)
    torch.cuda.synchronize()
    long_work(side)
    with torch.cuda.stream(side):
        late_tables.copy_(tables)
        late_lens.copy_(lens)
    status = kvcache.attend_pages(q, k, v, late_tables, late_lens, out, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and not status.any()
    long_work(side)
    with torch.cuda.stream(side):
        late_tables.fill_(-1)
    with pytest.raises(RuntimeError, match="block_tables entries must lie"):
        kvcache.attend_pages(q, k, v, late_tables, late_lens, out, stream=side.cuda_stream)
    with pytest.raises(RuntimeError, match="q must have shape|must be"):  # refusals name the argument on any stream
        kvcache.attend_pages(q[:, :, :64], k, v, tables, lens, out, stream=side)


def test_checked_calls_follow_the_current_stream():
    """A one-shot call whose tables the host checks comes behind the current stream's earlier work, on any stream."""
    from ztcp_b200 import kvcache

    kv = [700, 65, 900]
    k, v, tables, lens = ref.make_cache(kv, 64, 2, 128, BF16, 8)
    q = queries(3, 8, 128, BF16, 9)
    want, out, lse = torch.empty_like(q), torch.empty_like(q), torch.empty((3, 8), device=DEV)
    kvcache.attend_pages(q, k, v, tables, lens, want, lse=lse)
    mass, summed = torch.empty(tables.shape, device=DEV), torch.empty(tables.shape, device=DEV)
    kvcache.page_mass(q, k, tables, lens, lse, None, mass)
    late = torch.zeros_like(q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(DEV)
    long_work()
    out.fill_(7.0)
    summed.fill_(7.0)
    late.copy_(q)
    kvcache.attend_pages(late, k, v, tables, lens, out, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    late.zero_()
    torch.cuda.synchronize()
    long_work()
    summed.fill_(7.0)
    late.copy_(q)
    kvcache.page_mass(late, k, tables, lens, lse, None, summed, stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(summed, mass)


def test_one_shot_calls_in_a_graph():
    """A whole step of one-shot calls, host checks at their default, captured and replayed over new contents."""
    from ztcp_b200 import kvcache

    T, H, G, D, R = 64, 2, 4, 128, 64
    kv = [700, 65, 300]
    k, v, tables, lens = ref.make_cache(kv, T, H, D, BF16, 8, poison=False)
    k0, v0 = k.clone(), v.clone()
    fused = queries(3, H * G + 2 * H, D, BF16, 9)
    q, new_k, new_v = fused.split([H * G, H, H], dim=1)
    table = kvcache.rope_table(1024, R)
    slots = torch.empty(3, dtype=torch.int64, device=DEV)
    pos = torch.empty(3, dtype=torch.int32, device=DEV)
    rot, out = (torch.empty((3, H * G, D), dtype=BF16, device=DEV) for _ in range(2))
    lse, mass = torch.empty((3, H * G), device=DEV), torch.zeros(tables.shape, device=DEV)

    def set_inputs(n, seed):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        pos.copy_(lens - 1)
        slots.copy_(tables.gather(1, ((lens - 1) // T).long()[:, None])[:, 0].long() * T + (lens - 1) % T)
        fused.copy_(queries(3, H * G + 2 * H, D, BF16, seed))
        k.copy_(k0), v.copy_(v0), mass.zero_()

    def step():
        st = [kvcache.append_tokens(q, new_k, new_v, k, v, slots, pos, table, rot)]
        st.append(kvcache.attend_pages(rot, k, v, tables, lens, out, lse=lse))
        st.append(kvcache.page_mass(rot, k, tables, lens, lse, mass, mass, decay=0.5))
        sel = kvcache.select_cold_pages(mass, tables, lens, page_tokens=T, keep=3)
        return [out, lse, mass, k, v, *st, *sel]

    set_inputs(kv, 9)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for n, seed in ((kv, 9), ([640, 1, 129], 10)):
        set_inputs(n, seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        set_inputs(n, seed)
        for g, w in zip(got, step()):
            assert torch.equal(g, w)


@pytest.fixture()
def wait_limit():
    from ztcp_b200 import capi

    yield capi.load().ztcp_wait_limit
    capi.load().ztcp_wait_limit(0)


WAITING = [("attend", 1, 1, 64, None), ("attend", 1, 1, 576, 64), ("attend", 1, 40, 128, None), ("mass", 1, 1, 64, None),
           ("mass", 1, 40, 64, None), ("mass", 1, 90, 128, None), ("mass", 1, 20, 576, None)]  # by operator and max_q_len


@pytest.mark.parametrize("op,G,hint,D,rope", WAITING)
def test_waits_that_run_out(wait_limit, op, G, hint, D, rope):
    """With 65,536 sequences each CTA takes milliseconds to find its place on the line, for which its other warps wait:
    longer than a limit of a few microseconds.  The call reports it and ends; the next one is as ever."""
    from ztcp_b200 import kvcache

    n = 1 << 16
    g = torch.Generator(device=DEV).manual_seed(D)
    rnd = lambda *s: torch.randn(s, generator=g, device=DEV, dtype=torch.float32).to(BF16)  # noqa: E731
    k = rnd(64, 8, 1, D)
    v = None if rope else rnd(64, 8, 1, D)
    q = rnd(n, G, D)
    tables = torch.randint(0, 64, (n, 1), generator=g, device=DEV, dtype=torch.int32)
    lens = torch.ones(n, dtype=torch.int32, device=DEV)
    starts = torch.arange(n + 1, dtype=torch.int32, device=DEV)
    first = tables[:, 0].long()
    s = (q.double() * k[first, 0].double()).sum(-1) * D ** -0.5  # one key: its score is the log-sum-exp
    kw = dict(q_starts=starts, max_q_len=hint)
    if op == "attend":
        out, lse = torch.empty((n, G, D - (rope or 0)), dtype=BF16, device=DEV), torch.empty((n, G), device=DEV)
        call = kvcache.prepare_attend(q, k, v, tables, lens, out, lse=lse, rope_dim=rope or 0, **kw)
    else:
        out = torch.empty((n, 1), device=DEV)
        call = kvcache.prepare_page_mass(q, k, tables, lens, s.float(), None, out, **kw)
    for limit in (1000, 0):
        wait_limit(limit)
        out.fill_(9.0)
        status = call()
        torch.cuda.synchronize()
        assert bool((status == (kvcache.SEQ_TIMEOUT if limit else 0)).all())
    if op == "attend":
        values = k[first, 0, :, rope:] if rope else v[first, 0]
        assert torch.equal(out, values.expand_as(out))  # the weight is 1, and the sum
        assert bool(((lse - s).abs() <= (D + 8) * ref.U32 * (q.double().abs() * k[first, 0].double().abs()).sum(-1)).all())
    else:  # exp of a score's error and of its rounding
        bound = (D + 8) * ref.U32 * ((q.double().abs() * k[first, 0].double().abs()).sum(-1) * D ** -0.5 + 1)
        assert bool(((out - 1).abs() <= 2 * bound).all())


def test_many_sequences_without_rows():
    """The largest batch, of sequences without rows but the first and the last: the kernels' waits do not run out."""
    from ztcp_b200 import kvcache

    n, D = 1 << 21, 64
    k, v = (queries(64 * 8, 1, D, BF16, s).view(64, 8, 1, D) for s in (1, 2))
    starts = torch.ones(n + 1, dtype=torch.int32, device=DEV)
    starts[0], starts[-1] = 0, 301
    q = queries(301, 1, D, BF16, 3)
    tables = torch.zeros((n, 1), dtype=torch.int32, device=DEV)
    lens = torch.full((n,), 8, dtype=torch.int32, device=DEV)
    out, lse = torch.empty_like(q), torch.empty((301, 1), device=DEV)
    for hint in (1, 300):
        out.fill_(9.0)
        status = kvcache.attend_pages(q, k, v, tables, lens, out, lse=lse, q_starts=starts, max_q_len=hint, causal=False)
        assert not bool(status.any())
        want, wl, tol, ltol = ref.attend(cpu(q), cpu(k), cpu(v), cpu(tables[:2]), [8, 8], [1, 300], D ** -0.5, False)
        ref.assert_close(lse, wl, ltol, "lse")
        ref.assert_close(out, want, tol, "out")
        mass = torch.empty((n, 1), device=DEV)
        assert not bool(kvcache.page_mass(q, k, tables, lens, lse, None, mass, q_starts=starts, max_q_len=hint, causal=False).any())
        assert not bool(mass[1:-1].any())
        want, tol = ref.mass(cpu(q), cpu(k), cpu(tables[:2]), [8, 8], [1, 300], cpu(lse), None, 1.0, D ** -0.5, False)
        ref.assert_close(mass[[0, -1]], want, tol, "mass")


@pytest.mark.parametrize("limit", [1, 300, 2000, 6000, 20_000, 100_000])
def test_waits_that_may_run_out(wait_limit, limit):
    """Limits about what a call's waits take: all of a call's sequences report it, or none does and the results are right;
    calls with the default limit on the same workspaces are as before."""
    from ztcp_b200 import kvcache

    kv, q_lens = [3000, 70, 900, 1], [40, 1, 33, 1]
    calls = []
    for H, G, D, rope, m in ((2, 4, 128, None, 40), (2, 4, 64, None, 1), (1, 16, 576, 64, 1), (2, 8, 256, None, 1)):
        k, v, tables, lens = ref.make_cache(kv, 64, H, D, BF16, 5, mla=rope is not None)
        ql = q_lens if m > 1 else [1] * 4
        q = queries(sum(ql), H * G, D, BF16, 6)
        out, lse = torch.empty((q.shape[0], H * G, D - (rope or 0)), dtype=BF16, device=DEV), torch.empty(q.shape[:2], device=DEV)
        mass = torch.empty(tables.shape, device=DEV)
        kw = dict(q_starts=ref.starts_of(ql), max_q_len=m)
        attend = kvcache.prepare_attend(q, k, v, tables, lens, out, lse=lse, rope_dim=rope or 0, **kw)
        attend()
        fixed = lse.clone()
        calls += [(attend, (out, lse)), (kvcache.prepare_page_mass(q, k, tables, lens, fixed, None, mass, **kw), (mass,))]
    want = []
    for call, outs in calls:
        assert not call().any()
        want.append([t.clone() for t in outs])
    for _ in range(5):
        for (call, outs), w in zip(calls, want):
            wait_limit(limit)
            status = call().tolist()
            assert status in ([kvcache.SEQ_TIMEOUT] * 4, [0] * 4)
            if status[0] == 0:
                assert all(torch.equal(a, b) for a, b in zip(outs, w))
            wait_limit(0)
            assert not call().any() and all(torch.equal(a, b) for a, b in zip(outs, w))


# ---- attention weight per page ----------------------------------------------------------------------------------
def check_mass(kv, q_lens, T, H, G, D, dtype, *, causal=True, seed=1, decay=0.75, empty=True, bad=()):
    from ztcp_b200 import kvcache

    k, v, tables, lens = ref.make_cache(kv, T, H, D, dtype, seed, mla=True, extra_pages=2)
    for b, p in bad:
        tables[b, p] = -7
    q = queries(sum(q_lens), H * G, D, dtype, seed + 1)
    _, lse, _, _ = ref.attend(cpu(q), cpu(k), None, cpu(tables), kv, q_lens, D ** -0.5, causal)
    lse = lse.float().to(DEV)
    before = None if empty else torch.rand(tables.shape, device=DEV)
    out = torch.full(tables.shape, 9.0, device=DEV)
    status = kvcache.page_mass(q, k, tables, lens, lse, before, out, decay=decay, q_starts=ref.starts_of(q_lens),
                               max_q_len=max(max(q_lens), 1), causal=causal, check_block_table=False)
    torch.cuda.synchronize()
    want, tol = ref.mass(cpu(q), cpu(k), cpu(tables), kv, q_lens, cpu(lse), cpu(before), decay, D ** -0.5, causal)
    assert [s != 0 for s in status.tolist()] == [any(b == i for b, _ in bad) for i in range(len(kv))]
    ref.assert_close(out, want, tol, "mass")
    if before is not None:  # in place
        kvcache.page_mass(q, k, tables, lens, lse, before, before, decay=decay, q_starts=ref.starts_of(q_lens),
                          max_q_len=max(max(q_lens), 1), causal=causal, check_block_table=False)
        assert torch.equal(before, out)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=ids)
@pytest.mark.parametrize("T,H,G,D", [(64, 8, 4, 128), (16, 2, 1, 64), (5, 1, 3, 48), (100, 2, 8, 128), (256, 1, 4, 64),
                                     (64, 1, 16, 576), (64, 2, 4, 256), (128, 4, 2, 128), (8, 2, 4, 64)])
def test_mass_decode(dtype, T, H, G, D):
    check_mass([1, 64, 0, 300, 129], [1, 1, 1, 1, 1], T, H, G, D, dtype, empty=dtype == F16)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=ids)
@pytest.mark.parametrize("T,D", [(64, 128), (16, 64), (48, 128), (128, 64), (64, 112)])
@pytest.mark.parametrize("causal", [True, False])
def test_mass_window(dtype, T, D, causal):
    check_mass([200, 0, 70, 33, 513], [32, 3, 70, 0, 64], T, 2, 4, D, dtype, causal=causal, empty=False)


@pytest.mark.parametrize("H,G,D,T,q_max,batch", [(8, 4, 128, 64, 1, 40), (8, 4, 128, 64, 64, 6), (2, 8, 64, 16, 1, 40),
                                                  (4, 4, 64, 16, 100, 6), (1, 16, 576, 64, 2, 20)])
def test_mass_long_sequences(H, G, D, T, q_max, batch):
    from ztcp_b200 import kvcache

    kv, q_lens = ref.ragged(D + T, batch, 5000, q_max)
    kv = [n + 1500 for n in kv]
    q_lens = [max(1, m) for m in q_lens]
    k, _, tables, lens = ref.make_large_cache(kv, T, H, D, BF16, 9, True)
    q = queries(sum(q_lens), H * G, D, BF16, 8)
    lse = torch.empty(q.shape[:2], device=DEV)
    out = torch.empty((q.shape[0], H * G, D - 64 if D > 512 else D), dtype=BF16, device=DEV)
    starts = ref.starts_of(q_lens)
    kvcache.attend_pages(q, k, None if D > 512 else k.clone(), tables, lens, out, lse=lse, q_starts=starts,
                         max_q_len=q_max, rope_dim=64 if D > 512 else 0)
    before = torch.rand(tables.shape, device=DEV)
    mass = torch.empty_like(before)
    for _ in range(3):
        kvcache.page_mass(q, k, tables, lens, lse, before, mass, decay=0.5, q_starts=starts, max_q_len=q_max)
        torch.cuda.synchronize()
    want, tol = ref.mass_large(q, k, tables, kv, q_lens, lse, before, 0.5, D ** -0.5)
    ref.assert_close(mass, want, tol, "mass")


@pytest.mark.parametrize("G,D,n,q_len", [(128, 576, (1 << 24) + 130, 1), (64, 64, (1 << 25) + 77, 1), (16, 128, (1 << 27) + 5, 1),
                                         (128, 256, (1 << 24) + 300, 2)])
def test_mass_keys_far_before_the_window(G, D, n, q_len):
    """Keys whose distance to the window times the group passes 2^31 weigh what they should.  The table repeats a few
    pages, so that the pool is small and a page's weight follows from its contents."""
    from ztcp_b200 import kvcache

    T, pool = 64, 5
    g = torch.Generator().manual_seed(G)
    k = torch.randn((pool, T, 1, D), generator=g).to(BF16).to(DEV)
    q = queries(q_len, G, D, BF16, 3)
    P = -(-n // T)
    tables = (torch.arange(P, dtype=torch.int32, device=DEV) % pool)[None].contiguous()
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    scale = D ** -0.5
    s = torch.einsum("rgd,ptd->rgpt", q.double(), k[:, :, 0].double()) * scale
    # the log-sum-exp over the whole of the pages (the last one's unseen tokens are among 2^21 and more: left out)
    lse = (torch.logsumexp(s.flatten(2), 2) + torch.log(torch.tensor(n / (pool * T), dtype=torch.float64))).float()
    out = torch.empty((1, P), device=DEV)
    status = kvcache.page_mass(q, k, tables, lens, lse, None, out, q_starts=ref.starts_of([q_len]), max_q_len=q_len,
                               scale=scale, check_block_table=False)
    assert not status.any()
    size = torch.einsum("rgd,ptd->rgpt", q.double().abs(), k[:, :, 0].double().abs()) * scale
    w = torch.exp(s - lse.double()[..., None, None])
    e = (D + 3) * ref.U32 * size + 4 * ref.U32 * (s.abs() + lse.double().abs()[..., None, None]) + (T + q_len * G + 8) * ref.U32
    want, tol = w.sum((0, 1, 3)), (w * e).sum((0, 1, 3))
    whole = (n - q_len) // T  # pages that every row sees whole
    at = torch.arange(whole, device=DEV) % pool
    off = (out[0, :whole].double() - want[at]).abs() - tol[at] - 4 * ref.U32 * want[at]
    assert float(off.max()) <= 0, f"page {int(off.argmax())}: {float(off.max()):.3e} beyond the bound"
    last = torch.arange(whole * T, n, device=DEV)  # the others, token by token
    for p in range(whole, P):
        want_p = tol_p = 0.0
        for j in last[last // T == p].tolist():
            for i in range(q_len):
                if j <= n - q_len + i:
                    want_p += float(w[i, :, p % pool, j % T].sum())
                    tol_p += float((w * e)[i, :, p % pool, j % T].sum())
        assert abs(float(out[0, p]) - want_p) <= tol_p + 4 * ref.U32 * want_p


@pytest.mark.parametrize("q_len", [1, 12, 70])
def test_tiny_scale(q_len):
    """A scale near the smallest fp32 makes every score 0: every token weighs the same, masked ones nothing."""
    from ztcp_b200 import kvcache

    kv = [200, 70, 300]
    k, v, tables, lens = ref.make_cache(kv, 64, 2, 128, BF16, 5)
    q = queries(3 * q_len, 8, 128, BF16, 6)
    out, lse, status = run_attend(q, k, v, tables, lens, [q_len] * 3, scale=1e-39)
    want, wl, tol, ltol = ref.attend(cpu(q), cpu(k), cpu(v), cpu(tables), kv, [q_len] * 3, 1e-39)
    assert not status.any()
    ref.assert_close(lse, wl, ltol, "lse")
    ref.assert_close(out, want, tol, "out")
    mass = torch.empty(tables.shape, device=DEV)
    kvcache.page_mass(q, k, tables, lens, lse, None, mass, q_starts=ref.starts_of([q_len] * 3), max_q_len=q_len, scale=1e-39)
    want, tol = ref.mass(cpu(q), cpu(k), cpu(tables), kv, [q_len] * 3, cpu(lse), None, 1.0, 1e-39)
    ref.assert_close(mass, want, tol, "mass")


def one_key_scores(op, T, G, D, dtype, hint, rope, kind, n=4096):
    """Scores of n sequences of one token: (64-bit ones, the errors of the kernel's).  With one key the log-sum-exp is its
    score; a page's weight is the exponential of the score's error over a given log-sum-exp."""
    from ztcp_b200 import kvcache

    g = torch.Generator(device=DEV).manual_seed(D + G)
    rnd = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    q, key = rnd(n, G, D), rnd(n, D)
    if kind == "few bits":  # every product and every partial sum is exact
        q, key = q.sign() * 0.5 * (1 + (q.abs() > 1)), key.sign() * (1 + (key.abs() > 0.7))
    if kind == "one column":
        q = torch.zeros_like(q).scatter_(2, torch.randint(0, D, (n, G, 1), generator=g, device=DEV), 1.0) * q
    if kind == "positive":
        q, key = q.abs(), key.abs()
    q, key = q.to(dtype), key.to(dtype)
    k = torch.zeros((n, T, 1, D), dtype=dtype, device=DEV)
    k[:, 0, 0] = key
    tables = torch.arange(n, dtype=torch.int32, device=DEV)[:, None].contiguous()
    lens = torch.ones(n, dtype=torch.int32, device=DEV)
    kw = dict(q_starts=torch.arange(n + 1, dtype=torch.int32, device=DEV), max_q_len=hint, scale=1.0)
    s = torch.einsum("ngd,nd->ng", q.double(), key.double())
    if op == "attend":
        out, lse = torch.empty((n, G, D - (rope or 0)), dtype=dtype, device=DEV), torch.empty((n, G), device=DEV)
        kvcache.attend_pages(q, k, None if rope else k, tables, lens, out, lse=lse, rope_dim=rope or 0, **kw)
        return s, lse.double() - s
    errors, lse = [], s.float()
    for h in range(G):
        out = torch.empty((n, 1), device=DEV)
        kvcache.page_mass(q[:, h:h + 1].contiguous(), k, tables, lens, lse[:, h:h + 1].contiguous(), None, out, **kw)
        errors.append(torch.log(out[:, 0].double()) + lse[:, h].double() - s[:, h])
    return s, torch.stack(errors, 1)


SCORES = [("attend", 8, 4, 64, 1, None), ("attend", 8, 4, 128, 1, None), ("attend", 8, 4, 256, 1, None), ("attend", 8, 4, 576, 1, 64),
          ("attend", 8, 4, 128, 40, None), ("attend", 5, 4, 128, 1, None), ("attend", 5, 4, 320, 1, 16), ("attend", 5, 4, 576, 1, 64),
          ("mass", 8, 2, 64, 1, None), ("mass", 8, 2, 128, 1, None), ("mass", 8, 2, 128, 40, None), ("mass", 8, 2, 64, 90, None),
          ("mass", 8, 2, 128, 90, None), ("mass", 8, 2, 256, 1, None), ("mass", 8, 2, 256, 40, None), ("mass", 8, 2, 576, 1, None),
          ("mass", 8, 2, 576, 40, None), ("mass", 5, 2, 128, 1, None), ("mass", 5, 2, 576, 1, None)]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=ids)
@pytest.mark.parametrize("op,T,G,D,hint,rope", SCORES)
def test_exact_scores_stay_exact(op, T, G, D, hint, rope, dtype):
    """Where every product and partial sum is exact, so is the score: nothing is added to it for what other data would
    lose.  A page's weight under the score itself as log-sum-exp is then 1, to the bit.  Of the log-sum-exp, the rounded
    scale * log2(e) and ln 2 are at most a half step off each, the last fma another (with |score| each), and the sum of one
    weight, whose logarithm is added, two steps of 1."""
    for kind in ("few bits", "one column"):
        s, e = one_key_scores(op, T, G, D, dtype, hint, rope, kind)
        if op == "mass":
            exact = s.float().double() == s  # (all few-bit ones, and products of two 11-bit numbers)
            assert bool(exact.all()) and bool((e == 0).all())
        else:
            assert bool((e.abs() <= ref.U32 * (3 * s.abs() + 5)).all()), float(((e.abs() - 5 * ref.U32) / s.abs()).max()) / ref.U32


@pytest.mark.parametrize("D,hint,times", [(128, 1, 1.5), (128, 90, 1.5), (256, 40, 1.5), (576, 1, 1.5), (576, 40, 3)])
def test_score_loss_does_not_grow_with_the_columns(D, hint, times):
    """The tensor cores' accumulator drops the lowest bits of what it holds, for every product that it takes.  Positive
    data shows it: after each of n products it stands at an even share of the sum, so that the relative loss grows
    with n.  Page weights give an accumulator four products of 16 columns whatever the head_dim (eight with 32 rows of 576:
    about twice the loss), as at head_dim 64; one accumulator for 36 products loses 16 times as much."""
    base_s, base = one_key_scores("mass", 8, 2, 64, F16, hint, None, "positive")
    s, e = one_key_scores("mass", 8, 2, D, F16, hint, None, "positive")
    mean = lambda s, e: float(e.sum() / s.sum()) / ref.U32  # noqa: E731
    # (a half step for the sum of the parts and one for the exponent's rounding, in the mean at most)
    assert abs(mean(s, e)) <= times * abs(mean(base_s, base)) + 1


@pytest.mark.parametrize("kw,fits", [
    (dict(), True),
    # a page whose sums, 16 a segment and head, pass 2^31
    (dict(geom=(1 << 20, 4096, 16), n_seqs=1, max_pages=1), False),
    # sums of all sequences beyond any memory, their size beyond 64 bits in the second case
    (dict(geom=(1 << 15, 64, 64), n_seqs=1 << 12, max_pages=1 << 12), False),
    (dict(geom=(1 << 20, 1 << 9, 16), n_seqs=1 << 21, max_pages=1 << 11), False),
])
def test_mass_sums_that_do_not_fit(kw, fits):
    """Geometries, never launched here, whose segment sums pass 32 bits or a GPU's memory: they go to the kernel that needs
    no workspace."""
    from ztcp_b200 import capi, kvcache

    lib = kvcache._load()
    T, H, D = kw.pop("geom", (64, 8, 128))
    n, P = kw.get("n_seqs", 4), kw.get("max_pages", 16)
    c = kvcache._Cache(1 << 16, None, 0, 0, capi.geometry(T, H, D, 0, True), 1, 1 << 16, P, P, 1 << 16, n)
    q = kvcache._Queries(1 << 16, H * D * 4, D, 1 << 16, n, 4 * H, 64, 0.1, 1)
    size = lib.ztcp_page_mass_workspace_bytes(c, q)
    assert size > 16 if fits else size == 16


@pytest.mark.parametrize("dtype", [F16, BF16], ids=ids)
@pytest.mark.parametrize("H,G,D,T", [(1, 16, 576, 64), (1, 40, 576, 16), (2, 4, 256, 64), (1, 3, 320, 32), (2, 2, 176, 40), (2, 8, 128, 64)])
def test_mass_windows_of_wide_heads(H, G, D, T, dtype):
    """Windows of several chunks of rows at head dims beyond 128, latent pages among them, and of two 256-row chunks."""
    check_mass([200, 0, 70, 385], [32, 3, 70, 64], T, H, G, D, dtype, empty=False, bad=[(0, 1), (3, 2)])


@pytest.mark.parametrize("G,D", [(4, 128), (4, 64), (7, 112), (140, 128)])
def test_mass_items_of_one_and_two_row_tiles(G, D):
    """Many short items to a CTA, of one row tile and of two, of one chunk and of several, in any order: whichever group of
    warps an item's first step falls to."""
    from ztcp_b200 import kvcache

    kv, q_lens = ref.ragged(D + G, 300, 500, 64 if G < 100 else 3)
    kv = [n + 1 for n in kv]
    q_lens = [min(m, n) for m, n in zip(q_lens, kv)]
    k, v, tables, lens = ref.make_large_cache(kv, 16, 1, D, BF16, 9)
    q = queries(sum(q_lens), G, D, BF16, 8)
    lse, out = torch.empty(q.shape[:2], device=DEV), torch.empty_like(q)
    starts = ref.starts_of(q_lens)
    kvcache.attend_pages(q, k, v, tables, lens, out, lse=lse, q_starts=starts, max_q_len=64)
    before = torch.rand(tables.shape, device=DEV)
    mass = torch.empty_like(before)
    kvcache.page_mass(q, k, tables, lens, lse, before, mass, decay=0.5, q_starts=starts, max_q_len=64)
    want, tol = ref.mass_large(q, k, tables, kv, q_lens, lse, before, 0.5, D ** -0.5)
    ref.assert_close(mass, want, tol, "mass")


def test_mass_more_rows_than_tokens():
    check_mass([3, 10], [40, 200], 16, 1, 4, 64, F16)


@pytest.mark.parametrize("q_len", [1, 40])
def test_mass_bad_blocks(q_len):
    check_mass([200, 130, 64], [q_len] * 3, 64, 2, 4, 128, BF16, bad=[(0, 1), (1, 0)])


@pytest.mark.parametrize("H,G,T,q_lens", [(1, 272, 64, [3, 1, 2]), (2, 100, 16, [7, 2, 1]), (1, 8, 8, [90, 33, 32]), (2, 7, 32, [80, 36, 37])])
def test_mass_wide_chunks(H, G, T, q_lens):
    """Rows beyond a chunk of 256, groups wider than one, chunks that whole tokens do not fill, bad pages among them."""
    check_mass([300, 77, 140], q_lens, T, H, G, 64, BF16, bad=[(0, 1), (2, 0)])
    check_mass([300, 77, 140], q_lens, T, H, G, 128, F16, causal=False, empty=False)


def test_mass_sums_to_the_rows():
    """Without earlier weight, a sequence's pages add up to its rows times heads: every row's weights sum to 1."""
    from ztcp_b200 import kvcache

    kv, q_lens = [900, 64, 1], [40, 1, 1]
    k, v, tables, lens = ref.make_cache(kv, 64, 4, 128, BF16, 4)
    q = queries(42, 16, 128, BF16, 5)
    _, lse, _ = run_attend(q, k, v, tables, lens, q_lens)
    out = torch.empty(tables.shape, device=DEV)
    kvcache.page_mass(q, k, tables, lens, lse, None, out, q_starts=ref.starts_of(q_lens), max_q_len=40)
    for total, rows in zip(out.double().sum(1).tolist(), q_lens):
        # a weight is off by the errors of its score and of lse: scores of at most 2^4, 2^4 * 140 half steps each
        assert abs(total / (rows * 16) - 1) <= 2 * 16 * 140 * ref.U32


# ---- append -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16], ids=ids)
@pytest.mark.parametrize("n,Hq,H,D,R,interleaved,norm_from,weights,mla", [
    (1, 32, 8, 128, 128, False, 0, True, False),
    (37, 8, 2, 128, 64, True, 0, True, False),
    (300, 4, 1, 64, 64, False, 0, True, False),
    (5, 16, 1, 576, 64, False, 64, True, True),
    (5, 3, 2, 48, 16, True, 0, True, False),
    (9, 6, 3, 96, 96, False, 32, False, False),
    (4, 2, 2, 256, 256, False, 0, True, False),
    (4, 2, 1, 1024, 256, True, 0, True, False),
    (3, 5, 1, 80, 0, False, 16, True, False),
    (2, 1, 1, 16, 16, False, 0, True, True),
    (1001, 32, 8, 128, 128, False, 0, True, False),
    (1200, 32, 7, 128, 64, True, 0, True, False),
    (7001, 8, 2, 64, 32, False, 0, True, False),
    (701, 16, 1, 576, 64, True, 64, True, True),
    (2100, 7, 2, 256, 128, False, 0, True, False),
    (9001, 3, 1, 48, 0, False, 16, True, False),
    (600, 20, 2, 1024, 256, False, 0, True, False),
])
def test_append(dtype, n, Hq, H, D, R, interleaved, norm_from, weights, mla):
    from ztcp_b200 import kvcache

    g = torch.Generator().manual_seed(n * D)
    T, pages = 16, n // 16 + 3
    split = [Hq * D, H * D, 0 if mla else H * D]
    qkv = torch.randn((n, sum(split) + 8), generator=g).to(dtype)  # rows with a gap behind them
    q, k, v = (t.unflatten(1, (-1, D)) if t.shape[1] else None for t in qkv[:, :sum(split)].split(split, dim=1))
    qw, kw = ((1 + 0.2 * torch.randn(D - norm_from, generator=g)) if weights else None for _ in range(2))
    table = kvcache.rope_table(500, R, device="cpu") if R else None
    pos = torch.randint(0, 500, (n,), generator=g, dtype=torch.int32)
    slots = torch.randperm(pages * T, generator=g)[:n].clone()
    if n > 2:
        slots[1] = -1
    kp = torch.full((pages, T, H, D), 3.0, dtype=dtype, device=DEV)
    vp = None if mla else kp.clone()
    dq = qkv.to(DEV)
    dq, dk, dv = (t.unflatten(1, (-1, D)) if t.shape[1] else None for t in dq[:, :sum(split)].split(split, dim=1))
    qo = torch.empty((n, Hq, D), dtype=dtype, device=DEV)
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    status = kvcache.append_tokens(dq, dk, dv, kp, vp, dev(slots), dev(pos), dev(table), qo, q_weight=dev(qw),
                                   k_weight=dev(kw), norm_from=norm_from, eps=1e-5, interleaved=interleaved)
    assert not status.any()
    want, tol = ref.norm_rotate(q, qw, norm_from, 1e-5, table, pos, interleaved)
    ref.assert_close(qo, want, tol, "q")
    want, tol = ref.norm_rotate(k, kw, norm_from, 1e-5, table, pos, interleaved)
    written = slots >= 0
    ref.assert_close(kp.view(-1, H, D)[dev(slots[written])], want[written], tol[written], "k")
    rest = torch.ones(pages * T, dtype=torch.bool)
    rest[slots[written]] = False
    assert bool((kp.view(-1, H, D)[dev(rest)] == 3).all())
    if not mla:
        assert torch.equal(vp.view(-1, H, D)[dev(slots[written])].cpu(), v[written])
        assert bool((vp.view(-1, H, D)[dev(rest)] == 3).all())


def test_append_bad_slots_and_positions():
    from ztcp_b200 import kvcache

    n, H, D, T = 6, 2, 64, 16
    k, v, q = (queries(n, h, D, BF16, s) for h, s in ((H, 1), (H, 2), (4, 3)))
    kp = torch.full((2, T, H, D), 3.0, dtype=BF16, device=DEV)
    vp = kp.clone()
    table = kvcache.rope_table(50, 64)
    slots = torch.tensor([0, 32, -2, 5, 6, 1 << 40], dtype=torch.int64, device=DEV)
    pos = torch.tensor([0, 1, 2, 50, -1, 3], dtype=torch.int32, device=DEV)
    qo = torch.full_like(q, 9.0)
    status = kvcache.append_tokens(q, k, v, kp, vp, slots, pos, table, qo)
    bad = kvcache.SEQ_BAD_BLOCK
    assert status.tolist() == [0, bad, bad, bad, bad, bad]
    assert bool((qo[3:5] == 9).all())                       # a position outside the table: nothing is written
    assert not bool((qo[[0, 1, 2, 5]] == 9).all(-1).any())  # a slot outside the pool: the query only
    assert bool((kp.view(-1, H, D)[1:] == 3).all()) and not bool((kp.view(-1, H, D)[0] == 3).all())
    assert torch.equal(vp.view(-1, H, D)[0], v[0]) and bool((vp.view(-1, H, D)[1:] == 3).all())


def test_append_in_place_and_without_queries():
    from ztcp_b200 import kvcache

    n, H, D, T = 33, 2, 128, 64
    k, v, q = (queries(n, h, D, F16, s) for h, s in ((H, 1), (H, 2), (8, 3)))
    kp, vp = (torch.zeros((1, T, H, D), dtype=F16, device=DEV) for _ in range(2))
    table, pos = kvcache.rope_table(64, 128), torch.arange(n, dtype=torch.int32, device=DEV)
    slots = torch.arange(n, device=DEV)
    qo = torch.empty_like(q)
    kvcache.append_tokens(q, k, v, kp, vp, slots, pos, table, qo)
    kp2, vp2 = torch.zeros_like(kp), torch.zeros_like(vp)
    kvcache.append_tokens(q, k, v, kp2, vp2, slots, pos, table, q)
    assert torch.equal(q, qo) and torch.equal(kp, kp2)
    kp2.zero_()
    kvcache.append_tokens(None, k, v, kp2, vp2, slots, pos, table, None)
    assert torch.equal(kp, kp2) and torch.equal(vp, vp2)


# ---- eviction ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kv,T,keep,sink,recent", [
    ([640], 64, 4, 1, 1),
    ([0, 1, 64, 65, 1000, 5000, 4999], 16, 20, 2, 3),
    ([3000, 2000], 1, 100, 0, 1),
    ([500, 20], 16, 0, 0, 1),
    ([500, 20], 16, 1000, 3, 5),
    ([500, 48], 16, 2, 40, 40),
    ([70000], 16, 4000, 4, 8),
])
def test_select(kv, T, keep, sink, recent):
    from ztcp_b200 import kvcache

    P = max(-(-n // T) for n in kv) + 1
    g = torch.Generator().manual_seed(len(kv) * T)
    mass = torch.rand((len(kv), P), generator=g)
    mass[torch.rand(mass.shape, generator=g) < 0.4] = 0.25   # ties
    mass[torch.rand(mass.shape, generator=g) < 0.05] = float("nan")
    mass[torch.rand(mass.shape, generator=g) < 0.05] = float("inf")
    mass[torch.rand(mass.shape, generator=g) < 0.1] = 0.0
    mass[torch.rand(mass.shape, generator=g) < 0.1] = -0.0
    mass[torch.rand(mass.shape, generator=g) < 0.05] = -1.5
    tables = torch.randint(0, 1 << 20, (len(kv), P), generator=g, dtype=torch.int32)
    want = ref.select(mass.numpy(), tables, kv, T, keep, sink, recent)
    sel = kvcache.select_cold_pages(mass.to(DEV), tables.to(DEV), torch.tensor(kv, dtype=torch.int32, device=DEV),
                                    page_tokens=T, keep=keep, sink=sink, recent=recent)
    for got, exp, name in zip(sel, want, sel._fields):
        if name == "kept_mass":
            assert torch.equal(got.cpu().nan_to_num(nan=77.0), torch.tensor(exp).nan_to_num(nan=77.0)), name
        else:
            assert got.tolist() == exp, name
    assert not sel.status.any()


@pytest.mark.parametrize("n,keep", [(1024, 1), (1025, 500), (2048, 2047), (2049, 1), (4096, 4000), (4097, 100), (9001, 4500)])
def test_select_page_counts(n, keep):
    """Page counts about what a CTA holds at once; weights in a narrow range, all alike, and of every size."""
    from ztcp_b200 import kvcache

    g = torch.Generator().manual_seed(n)
    mass = torch.stack([1 + torch.rand(n, generator=g) / 4096, torch.full((n,), 0.5), torch.randn(n, generator=g).exp() ** 8])
    tables = torch.randint(0, 1 << 20, (3, n), generator=g, dtype=torch.int32)
    lens = [n, n - 1, n]
    want = ref.select(mass.numpy(), tables, lens, 1, keep, 1, 1)
    sel = kvcache.select_cold_pages(mass.to(DEV), tables.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
                                    page_tokens=1, keep=keep, sink=1, recent=1)
    for got, exp, name in zip(sel, want, sel._fields):
        assert torch.equal(got.cpu(), torch.tensor(exp, dtype=got.dtype).view(got.shape)), name


@pytest.mark.parametrize("n,P", [(511, 9), (512, 9), (513, 9), (1537, 3), (5000, 5), (70_000, 3)])
def test_select_many_sequences(n, P):
    """Batches about the size from which the cold lists' starts are added up beforehand, and far beyond."""
    from ztcp_b200 import kvcache

    g = torch.Generator().manual_seed(n)
    mass = torch.rand((n, P), generator=g)
    tables = torch.randint(0, 1 << 20, (n, P), generator=g, dtype=torch.int32)
    lens = torch.randint(0, P * 16 + 1, (n,), generator=g, dtype=torch.int32)
    want = ref.select(mass.numpy(), tables, lens.tolist(), 16, 2, 1, 1)
    sel = kvcache.select_cold_pages(mass.to(DEV), tables.to(DEV), lens.to(DEV), page_tokens=16, keep=2)
    for got, exp, name in zip(sel, want, sel._fields):
        assert torch.equal(got.cpu(), torch.tensor(exp, dtype=got.dtype).view(got.shape)), name
    assert not sel.status.any()


def test_select_takes_time_in_proportion():
    """Every sequence's place was once found by adding up all sequences' pages: 262,144 of them took 180 ms."""
    from ztcp_b200 import kvcache

    def time(n):
        mass, tables = torch.rand((n, 2), device=DEV), torch.zeros((n, 2), dtype=torch.int32, device=DEV)
        lens = torch.full((n,), 32, dtype=torch.int32, device=DEV)
        run = lambda: kvcache.select_cold_pages(mass, tables, lens, page_tokens=16, keep=1)  # noqa: E731
        run()
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        run()
        end.record()
        torch.cuda.synchronize()
        return begin.elapsed_time(end)

    assert time(1 << 18) < 60  # (a few ms)


def test_select_clamps_lengths():
    from ztcp_b200 import kvcache

    mass = torch.rand((2, 8), device=DEV)
    tables = torch.arange(16, dtype=torch.int32, device=DEV).view(2, 8)
    lens = torch.tensor([-3, 1 << 20], dtype=torch.int32, device=DEV)
    sel = kvcache.select_cold_pages(mass, tables, lens, page_tokens=16, keep=5)
    want = ref.select(mass.cpu().numpy(), tables.cpu(), [0, 128], 16, 5, 1, 1)
    assert sel.status.tolist() == [kvcache.SEQ_BAD_LENGTH] * 2
    assert sel.cold_blocks.tolist() == want[0] and sel.kept_tables.tolist() == want[3] and sel.kept_lens.tolist() == want[5]


# ---- together ---------------------------------------------------------------------------------------------------
def test_append_attend_mass_select_egress_ingress():
    """A serving loop over one layer: prompt chunks are appended and attended to, the pages with the least attention
    weight are chosen, encrypted from their pool slots and restored into fresh ones; attention over the compacted
    tables sees exactly the pages that stayed, over the restored ones what the codec gives back."""
    from ztcp_b200 import capi, codec, kvcache, workload

    T, H, Hq, D, R, pool = 64, 8, 32, 128, 64, 40
    prompts, q_scale = [700, 430], D ** -0.5
    g = torch.Generator().manual_seed(3)
    table = kvcache.rope_table(1024, R)
    w = (1 + 0.1 * torch.randn(D, generator=g)).to(DEV)
    kp, vp = (torch.zeros((pool, T, H, D), dtype=F16, device=DEV) for _ in range(2))
    tables = torch.randperm(pool, generator=g)[:2 * 12].view(2, 12).to(torch.int32).to(DEV)
    starts = ref.starts_of(prompts)
    n = sum(prompts)
    qkv = torch.randn((n, Hq + 2 * H, D), generator=g).to(F16).to(DEV)
    pos = torch.cat([torch.arange(m) for m in prompts])
    seq = torch.cat([torch.full((m,), b) for b, m in enumerate(prompts)])
    slots = tables.cpu()[seq, pos // T].long() * T + pos % T
    q = torch.empty((n, Hq, D), dtype=F16, device=DEV)
    st = kvcache.append_tokens(qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:], kp, vp, slots.to(DEV),
                               pos.to(torch.int32).to(DEV), table, q, q_weight=w, k_weight=w, interleaved=True)
    lens = torch.tensor(prompts, dtype=torch.int32, device=DEV)
    out, lse = torch.empty_like(q), torch.empty((n, Hq), device=DEV)
    st2 = kvcache.attend_pages(q, kp, vp, tables, lens, out, lse=lse, q_starts=starts, max_q_len=700)
    torch.cuda.synchronize()
    assert not st.any() and not st2.any()
    rows = torch.tensor([0, 5, 64, 699, 700, 1129])  # some rows against the plain form
    for r in rows.tolist():
        b, i = (0, r) if r < 700 else (1, r - 700)
        want, _, tol, _ = ref.attend(cpu(q[r:r + 1]), cpu(kp), cpu(vp), cpu(tables[b:b + 1]), [i + 1], [1], q_scale)
        ref.assert_close(out[r:r + 1], want, tol, f"row {r}")

    window = 16  # attention weight of each prompt's last rows
    pick = torch.cat([torch.arange(m - window, m) + s for m, s in zip(prompts, [0, 700])]).to(DEV)
    mass = torch.zeros(tables.shape, device=DEV)
    kvcache.page_mass(q[pick], kp, tables, lens, lse[pick], mass, mass, q_starts=ref.starts_of([window] * 2),
                      max_q_len=window)
    sel = kvcache.select_cold_pages(mass, tables, lens, page_tokens=T, keep=6, sink=1, recent=2)
    want = ref.select(mass.cpu().numpy(), tables.cpu(), prompts, T, 6, 1, 2)
    assert sel.cold_blocks.tolist() == want[0] and sel.kept_lens.tolist() == [700 - 5 * 64, 430 - 64]

    cold = int(sel.cold_starts[-1])
    assert cold == 6
    m = workload.session_material(5)
    keys = capi.keys(*m["key"], *m["mac_key"])
    hashes = torch.from_numpy(workload.token_hashes(24, 9)).to(DEV)[sel.cold_index[:cold].long()]
    blobs = torch.empty((cold, 98352), dtype=torch.uint8, device=DEV)
    kw = dict(rope_dim=64, tenant_id_hash=m["tenant"], model_id_hash=m["model"], layer_id=1, keys=keys)
    blocks = sel.cold_blocks[:cold].clone()
    codec.encode_pages(kp, vp, hashes, blobs, preset=1, rope_mode=1, expected_payload_bytes=98304, head_group_id=0,
                       base_sequence_nonce=1, block_table=blocks, **kw)

    # decode step over the compacted tables
    q1 = queries(2, Hq, D, F16, 12)
    o1 = torch.empty_like(q1)
    kvcache.attend_pages(q1, kp, vp, sel.kept_tables, sel.kept_lens, o1)
    want, _, tol, _ = ref.attend(cpu(q1), cpu(kp), cpu(vp), cpu(sel.kept_tables), sel.kept_lens.tolist(), [1, 1], q_scale)
    ref.assert_close(o1, want, tol, "compacted")

    # the cold pages come back into other pool pages
    free = [p for p in range(pool) if p not in set(tables.flatten().tolist())][:cold]
    back = torch.tensor(free, dtype=torch.int32, device=DEV)
    status, fail = codec.decode_pages(blobs, hashes, kp, vp, is_mla=False, block_table=back, **kw)
    codec.raise_for_status(status, fail)
    restored = tables.clone()
    restored.view(-1)[sel.cold_index[:cold].long()] = back
    kvcache.attend_pages(q1, kp, vp, restored, lens, o1)
    want, _, tol, _ = ref.attend(cpu(q1), cpu(kp), cpu(vp), cpu(restored), prompts, [1, 1], q_scale)
    ref.assert_close(o1, want, tol, "restored")


def test_cold_pages_through_the_staging_ring():
    """Selection -> store_cold -> load: the chosen pages, by sequence and page, come back as their own blobs' decode."""
    import test_gpu_hooks as hooks
    from ztcp_b200 import kvcache
    from ztcp_b200.cold_page_spec import ColdPageGeometry
    from ztcp_b200.hooks import CompactStagingRing, HiCachePageCodec
    from ztcp_b200.keyring import SessionKeyRing
    from ztcp_b200.session import ColdPageCodec

    ring = SessionKeyRing(b"h" * 32)
    hc = HiCachePageCodec(ColdPageCodec(ColdPageGeometry(num_tokens=64, num_kv_heads=8, head_dim=128, rope_dim=64), ring, DEV),
                          CompactStagingRing(32, 98352))
    k, v, tables, lens = ref.make_cache([640, 100, 300], 64, 8, 128, BF16, 3)
    k, v = k.nan_to_num(nan=0.0), v.nan_to_num(nan=0.0)  # unused rows of the pages are encrypted as well
    P = tables.shape[1]
    mass = torch.rand(tables.shape, generator=torch.Generator().manual_seed(4)).to(DEV)
    hashes = torch.arange(3 * P, device=DEV).view(3, P) * 7919 + 11
    sel = kvcache.select_cold_pages(mass, tables, lens, page_tokens=64, keep=3)
    n = int(sel.cold_starts[-1])
    assert n == 9
    view = hc.store_cold(sel, k, v, hashes, "tenant-h", "s", hooks._aad(ring.next_sequence_nonce("tenant-h", "s", n)))
    got_k, got_v = (torch.empty((n, 64, 8, 128), dtype=F16, device=DEV) for _ in range(2))
    assert hc.load(view, got_k, got_v, "tenant-h", "s", "model-h", 9).all()
    blocks = torch.tensor([int(tables[i // P, i % P]) for i in sel.cold_index[:n].tolist()], device=DEV)
    assert blocks.tolist() == sel.cold_blocks[:n].tolist()
    again = hc.store(k[blocks], v[blocks], hashes.view(-1)[sel.cold_index[:n].long()], "tenant-h", "s",
                     hooks._aad(ring.next_sequence_nonce("tenant-h", "s", n)))
    want_k, want_v = torch.empty_like(got_k), torch.empty_like(got_v)
    assert hc.load(again, want_k, want_v, "tenant-h", "s", "model-h", 9).all()
    assert torch.equal(got_k, want_k) and torch.equal(got_v, want_v)
    with pytest.raises(RuntimeError, match="page_token_hashes must have the block tables' shape"):
        hc.store_cold(sel, k, v, hashes[:2], "tenant-h", "s", hooks._aad(1))
    with pytest.raises(RuntimeError, match="block_tables entries must lie in"):
        hc.store_cold(sel, k[:1], v[:1], hashes, "tenant-h", "s", hooks._aad(1))
    none = kvcache.select_cold_pages(mass, tables, lens, page_tokens=64, keep=100)
    with pytest.raises(RuntimeError, match="no cold page"):
        hc.store_cold(none, k, v, hashes, "tenant-h", "s", hooks._aad(1))


def test_store_cold_waits_for_the_selections_stream():
    """A selection on another stream, still to run when store_cold is called; selections that it must not follow."""
    import test_gpu_hooks as hooks
    from ztcp_b200 import kvcache
    from ztcp_b200.cold_page_spec import ColdPageGeometry
    from ztcp_b200.hooks import CompactStagingRing, HiCachePageCodec
    from ztcp_b200.keyring import SessionKeyRing
    from ztcp_b200.session import ColdPageCodec

    ring = SessionKeyRing(b"h" * 32)
    hc = HiCachePageCodec(ColdPageCodec(ColdPageGeometry(num_tokens=64, num_kv_heads=8, head_dim=128, rope_dim=64), ring, DEV),
                          CompactStagingRing(32, 98352))
    k, v, tables, lens = ref.make_cache([640, 100, 300], 64, 8, 128, BF16, 3, poison=False)
    P = tables.shape[1]
    mass = torch.rand(tables.shape, generator=torch.Generator().manual_seed(4)).to(DEV)
    hashes = torch.arange(3 * P, device=DEV).view(3, P) * 7919 + 11
    args = ("tenant-h", "s")
    sel = kvcache.select_cold_pages(mass, tables, lens, page_tokens=64, keep=3)
    want_starts, n = sel.cold_starts.clone(), int(sel.cold_starts[-1])
    want = hc.store_cold(sel, k, v, hashes, *args, hooks._aad(ring.next_sequence_nonce("tenant-h", "s", n)))
    want_k, want_v = (torch.empty((n, 64, 8, 128), dtype=F16, device=DEV) for _ in range(2))
    assert hc.load(want, want_k, want_v, *args, "model-h", 9).all()
    side = torch.cuda.Stream(DEV)
    for stream in (side, side.cuda_stream):
        torch.cuda.synchronize()
        long_work(side)
        late = kvcache.select_cold_pages(mass, tables, lens, page_tokens=64, keep=3, stream=side)
        view = hc.store_cold(late, k, v, hashes, *args, hooks._aad(ring.next_sequence_nonce("tenant-h", "s", n)), stream=stream)
        got_k, got_v = torch.empty_like(want_k), torch.empty_like(want_v)
        assert hc.load(view, got_k, got_v, *args, "model-h", 9).all()
        assert torch.equal(late.cold_starts, want_starts) and torch.equal(got_k, want_k) and torch.equal(got_v, want_v)

    def refuse(match, **kw):
        with pytest.raises(RuntimeError, match=match):
            hc.store_cold(sel._replace(**kw), k, v, hashes, *args, hooks._aad(1))

    refuse("kv_len lies outside its block table", status=torch.tensor([0, kvcache.SEQ_BAD_LENGTH, 0], dtype=torch.int32, device=DEV))
    refuse("cold_index entries must lie in", cold_index=sel.cold_index + 3 * P)
    refuse("cold_index entries must lie in", cold_index=sel.cold_index - 3 * P)
    refuse("cold_starts must end with at most", cold_starts=sel.cold_starts + 3 * P)
    refuse("cold_starts must end with at most", cold_starts=sel.cold_starts - 3 * P)
    live = hc.ring.free_slots
    refuse("block_tables entries must lie in", cold_blocks=sel.cold_blocks + k.shape[0])
    assert hc.ring.free_slots == live
