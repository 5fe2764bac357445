"""Plain 64-bit forms of the paged-pool operators, and bounds on a 32-bit evaluation of them, for the tests."""
from __future__ import annotations

import random

import numpy as np
import torch

U32 = 2.0 ** -24  # half a step of fp32


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def make_cache(kv_lens, T, H, D, dtype, seed=0, mla=False, spare=3, poison=True, device="cuda", extra_pages=0):
    """A pool with shuffled block tables for sequences of these lengths.  Everything that no sequence holds -- unused
    pages, rows past a sequence's end -- is NaN when ``poison``; unused table entries point far outside the pool."""
    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // T) for n in kv_lens]
    pool = sum(pages) + spare
    order = torch.randperm(pool, generator=g).to(torch.int32)
    P = max(max(pages), 1) + extra_pages
    tables = torch.full((len(kv_lens), P), 2**31 - 1, dtype=torch.int32)
    fill = float("nan") if poison else 0.0
    k = torch.full((pool, T, H, D), fill, dtype=dtype)
    v = None if mla else torch.full((pool, T, H, D), fill, dtype=dtype)
    at = 0
    for b, n in enumerate(kv_lens):
        tables[b, :pages[b]] = order[at:at + pages[b]]
        at += pages[b]
        for p in range(pages[b]):
            rows = min(T, n - p * T)
            k[tables[b, p], :rows] = torch.randn((rows, H, D), generator=g).to(dtype)
            if v is not None:
                v[tables[b, p], :rows] = torch.randn((rows, H, D), generator=g).to(dtype)
    dev = lambda t: None if t is None else t.to(device)  # noqa: E731
    return dev(k), dev(v), dev(tables), torch.tensor(kv_lens, dtype=torch.int32, device=device)


def starts_of(q_lens, device="cuda"):
    return torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32, device=device)


def gather_rows(pool, table, n, bad=()):
    """Tokens [0, n) of one sequence: rows [n, H, D] in 64 bits, zeros for pages in `bad` (CPU tensors)."""
    T, H, D = pool.shape[1:]
    rows = torch.zeros((n, H, D), dtype=torch.float64)
    for p in range(-(-n // T)):
        if p not in bad:
            m = min(T, n - p * T)
            rows[p * T:p * T + m] = pool[int(table[p]), :m].double()
    return rows


def attend(q, k_pool, v_pool, tables, kv_lens, q_lens, scale, causal=True, rope_dim=0, pool_pages=None):
    """(out, lse, bound of out, bound of lse) in 64 bits; all inputs on the CPU.

    The bounds: with u the half step of the 16-bit type, A = sum_j w_j |v_j| and e a bound on the error of a weight,
    |out error| <= u |out| (its rounding) + u A (the weights' rounding before the second product) + 2 e A.
    e: a score is a sum of D exact products, so at most D half steps of sum |q_i k_i| off, and three roundings more
    for the scale, the maximum's subtraction and the exponential's 2 units; the sum l of n weights adds n half steps."""
    u = half_step(q.dtype)
    T, H, D = k_pool.shape[1:]
    G = q.shape[1] // H
    dv = D - (rope_dim if v_pool is None else 0)
    pool_pages = k_pool.shape[0] if pool_pages is None else pool_pages
    out = torch.zeros((q.shape[0], q.shape[1], dv), dtype=torch.float64)
    tol = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], float("-inf"), dtype=torch.float64)
    ltol = torch.zeros_like(lse)
    row = 0
    for b, (n, m) in enumerate(zip(kv_lens, q_lens)):
        bad = [p for p in range(-(-n // T)) if not 0 <= int(tables[b, p]) < pool_pages]
        keys = gather_rows(k_pool, tables[b], n, bad)
        vals = keys[..., D - dv:] if v_pool is None else gather_rows(v_pool, tables[b], n, bad)
        gone = torch.isin(torch.arange(n) // T, torch.tensor(bad, dtype=torch.long))
        for i in range(m):
            seen = min(n, max(0, n - m + i + 1)) if causal else n
            at = torch.nonzero(~gone[:seen]).flatten()
            if at.numel():
                for h in range(q.shape[1]):
                    qv, kv = q[row + i, h].double(), keys[at, h // G]
                    s = kv @ qv * scale
                    size = float((kv.abs() @ qv.abs()).max()) * scale
                    l = torch.logsumexp(s, 0)
                    w = torch.exp(s - l)
                    out[row + i, h] = w @ vals[at, h // G]
                    a = w @ vals[at, h // G].abs()
                    e = (D + 3) * U32 * size + float(s.abs().max()) * 4 * U32 + (at.numel() + 8) * U32
                    tol[row + i, h] = u * out[row + i, h].abs() + (u + 2 * e) * a + torch.finfo(q.dtype).tiny
                    lse[row + i, h] = l
                    ltol[row + i, h] = e + 4 * U32 * abs(float(l))
        row += m
    return out, lse, tol, ltol


def mass(q, k_pool, tables, kv_lens, q_lens, lse, before, decay, scale, causal=True):
    """(out_mass, bound) in 64 bits; all inputs on the CPU.  A weight's relative error: that of its score, as in
    ``attend``, plus the rounding of lse; a page sums positive weights, with at most a half step per addition."""
    T, H, D = k_pool.shape[1:]
    G = q.shape[1] // H
    P = tables.shape[1]
    out = torch.zeros((len(kv_lens), P), dtype=torch.float64)
    tol = torch.zeros_like(out)
    row = 0
    for b, (n, m) in enumerate(zip(kv_lens, q_lens)):
        pages = -(-n // T)
        bad = [p for p in range(pages) if not 0 <= int(tables[b, p]) < k_pool.shape[0]]
        keys = gather_rows(k_pool, tables[b], n, bad)
        gone = torch.isin(torch.arange(n) // T, torch.tensor(bad, dtype=torch.long))
        for i in range(m):
            seen = min(n, max(0, n - m + i + 1)) if causal else n
            at = torch.nonzero(~gone[:seen]).flatten()
            for h in range(q.shape[1]):
                l = lse[row + i, h].double()
                if not at.numel() or l == float("-inf"):
                    continue
                qv, kv = q[row + i, h].double(), keys[at, h // G]
                s = kv @ qv * scale
                w = torch.exp(s - l)
                e = ((D + 3) * U32 * (kv.abs() @ qv.abs()) * scale + 4 * U32 * (s.abs() + l.abs())
                     + (T + m * q.shape[1] + 8) * U32)
                out[b].index_add_(0, at // T, w)
                tol[b].index_add_(0, at // T, w * e)
        row += m
        if before is not None:
            out[b, :pages] += decay * before[b, :pages].double()
        tol[b] += 4 * U32 * out[b].abs()
    return out, tol


def select(mass, tables, kv_lens, T, keep, sink, recent):
    """The outputs of select_cold_pages as lists: (blocks, index, starts, kept tables, kept mass, kept lens)."""
    B, P = mass.shape
    blocks, index, starts, kt, km, kl = [], [], [0], [], [], []
    for b, n in enumerate(kv_lens):
        pages = -(-n // T)
        count = max(0, min(pages - keep, pages - sink - recent))
        key = lambda p: (1, 0.0, p) if np.isnan(mass[b, p]) else (0, float(mass[b, p]), p)  # noqa: E731
        cold = sorted(sorted(range(sink, max(sink, pages - recent)), key=key)[:count])
        stay = [p for p in range(pages) if p not in cold]
        blocks += [int(tables[b, p]) for p in cold]
        index += [b * P + p for p in cold]
        starts.append(len(blocks))
        kt.append([int(tables[b, p]) for p in stay] + [-1] * (P - len(stay)))
        km.append([float(mass[b, p]) for p in stay] + [0.0] * (P - len(stay)))
        kl.append(n - count * T)
    tail = [-1] * (B * P - len(blocks))
    return blocks + tail, index + tail, starts, kt, km, kl


def norm_rotate(x, weight, norm_from, eps, table, positions, interleaved):
    """(y, bound) of one [n, heads, D] tensor in 64 bits (CPU): a norm of D columns is at most D/2 + 4 half steps of
    its factor off, a rotation three more of |a cos| + |b sin|, and the result is rounded to the input's type."""
    u, D = half_step(x.dtype), x.shape[-1]
    y = x.double().clone()
    if weight is not None:
        f = y[..., norm_from:]
        y[..., norm_from:] = f / torch.sqrt((f ** 2).mean(-1, keepdim=True) + eps) * weight.double()
    size = y.abs().clone()
    if table is not None:
        R = table.shape[1]
        cs = table.double()[positions.long()][:, None]
        cos, sin = cs[..., :R // 2], cs[..., R // 2:]
        a, b = (y[..., 0:R:2], y[..., 1:R:2]) if interleaved else (y[..., :R // 2], y[..., R // 2:R])
        a, b = a.clone(), b.clone()
        lo, hi = a * cos - b * sin, b * cos + a * sin
        slo, shi = (a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()
        for t, p, q in ((y, lo, hi), (size, slo, shi)):
            if interleaved:
                t[..., 0:R:2], t[..., 1:R:2] = p, q
            else:
                t[..., :R // 2], t[..., R // 2:R] = p, q
    return y, u * y.abs() + (D / 2 + 8) * U32 * size + torch.finfo(x.dtype).tiny


def assert_close(got, want, tol, what):
    got = got.double().cpu()
    assert got.shape == want.shape, what
    empty = torch.isinf(want)
    assert torch.equal(got[empty], want[empty]), f"{what}: infinities differ"
    off = (got - want).abs()[~empty]
    worst = (off - tol[~empty]).max() if off.numel() else torch.tensor(0.0)
    assert bool((off <= tol[~empty]).all()), f"{what}: {float(worst):.3e} beyond the bound (largest error {float(off.max()):.3e})"


def ragged(seed, batch, kv_max, q_max):
    r = random.Random(seed)
    kv = [r.randint(0, kv_max) for _ in range(batch)]
    return kv, [r.randint(0, min(q_max, max(n, 1))) for n in kv]


def dense_sequence(pool, table, n):
    """Tokens [0, n) of one sequence, on the pool's device: [n, H, D]."""
    T = pool.shape[1]
    at = torch.arange(n, device=pool.device)
    return pool[table[at // T].long(), at % T]


def attend_large(q, k_pool, v_pool, tables, kv_lens, q_lens, scale, rope_dim=0):
    """``attend`` (causal) for long sequences: the same numbers and bounds, on the inputs' device, a head at a time."""
    u, D = half_step(q.dtype), k_pool.shape[3]
    H = k_pool.shape[2]
    G = q.shape[1] // H
    dv = D - (rope_dim if v_pool is None else 0)
    out = torch.zeros((q.shape[0], q.shape[1], dv), dtype=torch.float64, device=q.device)
    tol, lse = torch.zeros_like(out), torch.full(q.shape[:2], float("-inf"), dtype=torch.float64, device=q.device)
    ltol = torch.zeros_like(lse)
    row = 0
    for b, (n, m) in enumerate(zip(kv_lens, q_lens)):
        if n and m:
            keys = dense_sequence(k_pool, tables[b], n).double()
            vals = keys[..., D - dv:] if v_pool is None else dense_sequence(v_pool, tables[b], n).double()
            hidden = torch.arange(n, device=q.device)[None] > (torch.arange(m, device=q.device) + n - m)[:, None]
            for h in range(q.shape[1]):
                qv, kv, vv = q[row:row + m, h].double(), keys[:, h // G], vals[:, h // G]
                s = (qv @ kv.T * scale).masked_fill(hidden, float("-inf"))
                size = (qv.abs() @ kv.abs().T * scale).masked_fill(hidden, 0).amax(1)
                l = torch.logsumexp(s, 1)
                w = torch.exp(s - l[:, None])
                e = (D + 3) * U32 * size + s.masked_fill(hidden, 0).abs().amax(1) * 4 * U32 + (n + 8) * U32
                o = w @ vv
                out[row:row + m, h] = o
                tol[row:row + m, h] = u * o.abs() + (u + 2 * e)[:, None] * (w @ vv.abs()) + torch.finfo(q.dtype).tiny
                lse[row:row + m, h] = l
                ltol[row:row + m, h] = e + 4 * U32 * l.abs()
        row += m
    return out.cpu(), lse.cpu(), tol.cpu(), ltol.cpu()


def mass_large(q, k_pool, tables, kv_lens, q_lens, lse, before, decay, scale):
    """``mass`` (causal) for long sequences, on the inputs' device."""
    T, H, D = k_pool.shape[1:]
    G = q.shape[1] // H
    out = torch.zeros(tables.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    row = 0
    for b, (n, m) in enumerate(zip(kv_lens, q_lens)):
        page = torch.arange(n, device=q.device) // T
        if n and m:
            keys = dense_sequence(k_pool, tables[b], n).double()
            hidden = torch.arange(n, device=q.device)[None] > (torch.arange(m, device=q.device) + n - m)[:, None]
            for h in range(q.shape[1]):
                qv, kv, l = q[row:row + m, h].double(), keys[:, h // G], lse[row:row + m, h, None].double()
                s = (qv @ kv.T * scale).masked_fill(hidden, float("-inf"))
                w = torch.exp(s - l).nan_to_num(nan=0.0)
                e = ((D + 3) * U32 * (qv.abs() @ kv.abs().T) * scale + 4 * U32 * (s.masked_fill(hidden, 0).abs() + l.abs().nan_to_num(posinf=0.0))
                     + (T + m * q.shape[1] + 8) * U32)
                out[b].index_add_(0, page, w.sum(0))
                tol[b].index_add_(0, page, (w * e).sum(0))
        if before is not None:
            out[b, :-(-n // T)] += decay * before[b, :-(-n // T)].double()
        tol[b] += 4 * U32 * out[b].abs()
        row += m
    return out.cpu(), tol.cpu()


def make_large_cache(kv_lens, T, H, D, dtype, seed, mla=False):
    """``make_cache`` without NaN in the unused rows, made on the GPU."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = [-(-n // T) for n in kv_lens]
    pool = sum(pages) + 2
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    tables = torch.full((len(kv_lens), max(pages)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(pages):
        tables[b, :n] = order[at:at + n]
        at += n
    k, v = (torch.randn((pool, T, H, D), generator=g, device="cuda").to(dtype) for _ in range(2))
    return k, None if mla else v, tables, torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
