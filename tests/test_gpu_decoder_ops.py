"""GPU checks of the decoder operators (norm, page tables, rope + cache write, paged attention)
against plain implementations in 64 bits.

Bars, from the arithmetic. bf16 keeps 8 significant bits, so rounding to it moves a value
by at most 2^-8 of it (1 + 2^-8 lies halfway); e4m3 within 2^-4, or half of its
smallest step (2^-10, times the scale). The kernels' fp32 sums over at most 16384 terms are
allowed 1e-5 of the magnitudes summed. Attention rounds each probability to bf16 before the
product with V, so an output may be off by 2^-8 of sum(p |v|) / sum(p) besides its own rounding;
a score's fp32 sum of D products is allowed D * 2^-24 of sum |q k| (lse moves by no more than the
largest score error), and the exponentials and the logarithm 2^-20 of 1 + |lse|. Whole numbers are equal.
"""

import math
import random
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from vllm_ascend_hust_latchmoe_b200 import _lib
from vllm_ascend_hust_latchmoe_b200 import decoder_ops as ops

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]
BF16 = 2.0 ** -8
SUMS = 1e-5


def _gen(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def _bf16(g, *shape, std=1.0):
    return (torch.randn(*shape, device=g.device, generator=g) * std).to(torch.bfloat16)


def _within(got, want, bound):
    got, want = got.double(), want.double()
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), (got - want).abs().max().item(), bound.max().item())


# ------------------------------------------------------------------------------------- norm
def _norm64(x, residual, weight, eps):
    z = x.double() + (residual.double() if residual is not None else 0)
    return z, z / ((z * z).mean(1, keepdim=True) + eps).sqrt() * weight.double()


@pytest.mark.parametrize("T,H", [(1, 1), (1, 8), (3, 64), (2, 1000), (5, 1001), (16, 2048),
                                 (300, 2880), (149, 4096), (7, 5120), (33, 7168), (2, 16384),
                                 (1, 16383), (4093, 2048), (0, 64)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_norm_bf16(cuda, T, H, with_residual):
    g = _gen(cuda, T * 17 + H)
    x, w = _bf16(g, T, H, std=3.0), _bf16(g, H, std=0.3) + 1
    r = _bf16(g, T, H, std=20.0) if with_residual else None
    out, kept = torch.empty_like(x), torch.empty_like(x) if with_residual else None
    ops.add_rms_norm(x, w, 1e-6, residual=r, residual_out=kept, out=out)
    z, y = _norm64(x, r, w, 1e-6)
    _within(out, y, (BF16 + SUMS) * y.abs())
    if with_residual:
        _within(kept, z, BF16 * z.abs() + 2.0 ** -24 * (x.double().abs() + r.double().abs()))


@pytest.mark.parametrize("T,H,group", [(1, 64, 0), (16, 2048, 0), (16, 2048, 128), (5, 1001, 0),
                                       (3, 96, 32), (130, 4096, 128), (7, 7168, 128),
                                       (2, 16384, 64), (9, 2880, 0), (4, 8192, 8192),
                                       (3, 2880, 96), (5, 2304, 288)])
def test_norm_e4m3(cuda, T, H, group):
    g = _gen(cuda, T * 31 + H + group)
    x, r, w = _bf16(g, T, H), _bf16(g, T, H, std=5.0), _bf16(g, H, std=0.3) + 1
    x[:, H // 2] = 300.0  # an outlying column sets its group's scale
    out = torch.empty(T, H, dtype=torch.float8_e4m3fn, device=cuda)
    scales = torch.empty(T, H // group if group else 1, device=cuda)
    kept = torch.empty_like(x)
    ops.add_rms_norm(x, w, 1e-6, residual=r, residual_out=kept, out_fp8=out, scales=scales,
                     group_size=group)
    _, y = _norm64(x, r, w, 1e-6)
    want = y.view(T, -1, group or H).abs().amax(-1).clamp(min=1e-12) / 448
    _within(scales, want, SUMS * want)
    s = scales.double().repeat_interleave(group or H, dim=1)
    _within(out.double() * s, y, (2.0 ** -4 + SUMS) * y.abs() + (2.0 ** -10 + SUMS) * s)


def test_norm_zero_rows_and_special_values(cuda):
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device=cuda)
    x[1, 3] = math.inf
    x[2, 3] = math.nan
    x[3] = 3e38  # the sum of squares overflows fp32: 1 / sqrt(inf) = 0
    w = torch.ones(256, dtype=torch.bfloat16, device=cuda)
    out = torch.empty_like(x)
    ops.add_rms_norm(x, w, 1e-6, out=out)
    assert (out[0] == 0).all()
    assert out[1].isnan()[3] and (out[1][:3] == 0).all()
    assert out[2].isnan().all()
    assert (out[3] == 0).all()
    out8 = torch.empty(4, 256, dtype=torch.float8_e4m3fn, device=cuda)
    scales = torch.empty(4, 2, device=cuda)
    ops.add_rms_norm(x[:1].expand(4, 256).contiguous(), w, 1e-6, out_fp8=out8, scales=scales, group_size=128)
    assert (out8.float() == 0).all()
    _within(scales / (1e-12 / 448), torch.ones_like(scales), SUMS)


@pytest.mark.parametrize("T,H,pad", [(33, 2048, 64), (33, 2048, 3), (5, 1000, 1), (1, 2048, 0)])
def test_norm_strides_and_in_place(cuda, T, H, pad):
    g = _gen(cuda, H + pad)
    wide = _bf16(g, T, H + pad)
    x = wide[:, pad:] if pad % 2 else wide[:, :H]  # an odd offset: rows that no wide load fits
    r, w = _bf16(g, T, H, std=4.0), _bf16(g, H)
    out = torch.full((T, H + 2 * pad), 7.0, dtype=torch.bfloat16, device=cuda)
    z, y = _norm64(x, r, w, 1e-5)
    before = wide.clone()
    ops.add_rms_norm(x, w, 1e-5, residual=r, residual_out=r, out=out[:, :H])
    _within(out[:, :H], y, (BF16 + SUMS) * y.abs())
    assert (out[:, H:] == 7.0).all() and torch.equal(wide, before)
    _within(r, z, BF16 * z.abs() + 1e-6 * z.abs().max())
    # the residual stream into x's own storage, and y over x
    x2, r2 = _bf16(g, T, H), _bf16(g, T, H)
    z, y = _norm64(x2, r2, w, 1e-5)
    out2 = torch.empty_like(x2)
    ops.add_rms_norm(x2, w, 1e-5, residual=r2, residual_out=x2, out=out2)
    _within(out2, y, (BF16 + SUMS) * y.abs())
    _within(x2, z, BF16 * z.abs() + 1e-6 * z.abs().max())


# ------------------------------------------------------------------------------ page tables
def _tables_by_hand(cached, new, page, tables, free, count, T):
    seq, cu, pos, slots = [], [0], [], []
    err = 0
    dry = False
    taken = 0
    for b, (c, n) in enumerate(zip(cached, new)):
        have, total = -(-c // page), -(-(c + n) // page)
        ok = total <= len(tables[b])
        if not ok:
            err = 5
        else:
            taken += total - have
            if total > have and taken > count:
                ok, err = False, 5
        if ok:
            for i in range(have, total):
                tables[b][i] = free[count - 1 - (taken - total + i)]
        for t in range(n):
            pos.append(c + t)
            slots.append(tables[b][(c + t) // page] * page + (c + t) % page if ok else -1)
        seq.append(c + n if ok else c)
        cu.append(cu[-1] + n)
        if ok and total > have:
            dry = count - taken
    left = count if dry is False else dry
    return seq, cu, pos + [0] * (T - len(pos)), slots + [-1] * (T - len(slots)), left, err


def _tables_case(cuda, cached, new, page, width, spare=5, pad=7, count=None, in_place=False, stride=0):
    rng = random.Random(len(cached) * 7 + page)
    B = len(cached)
    have = [-(-c // page) for c in cached]
    pool = list(range(sum(have) + sum(-(-(c + n) // page) - h for c, n, h in zip(cached, new, have)) + spare))
    rng.shuffle(pool)
    tables = [[-1] * width for _ in range(B)]
    at = 0
    for b in range(B):
        for i in range(have[b]):
            tables[b][i] = pool[at]
            at += 1
    free = pool[at:]
    count = len(free) if count is None else count
    T = sum(new) + pad

    def ints(v, dtype=torch.int32):
        return torch.tensor(v, dtype=dtype, device=cuda)

    dt = torch.full((B, width + stride), -9, dtype=torch.int32, device=cuda)[:, :width]
    if B:
        dt.copy_(ints(tables).view(B, width))
    dc, dn, dfree, dcount = ints(cached), ints(new), ints(free or [0]), ints([count])
    seq = dc if in_place else torch.full((B,), -5, dtype=torch.int32, device=cuda)
    cu, pos = ints([-5] * (B + 1)), ints([-5] * T)
    slots, err = ints([-5] * T, torch.int64), ints([0])
    left = dcount if in_place else ints([-5])
    ops.build_page_tables(dc, dn, page, dt, dfree, dcount, seq_lens=seq, cu_q=cu, positions=pos,
                          slot_mapping=slots, free_count_out=left, err_word=err)
    w_seq, w_cu, w_pos, w_slots, w_left, w_err = _tables_by_hand(cached, new, page, tables, free, count, T)
    assert seq.tolist() == w_seq and cu.tolist() == w_cu
    assert pos.tolist() == w_pos and slots.tolist() == w_slots
    assert dt.tolist() == tables
    assert (left.item(), err.item()) == (w_left, w_err)


@pytest.mark.parametrize("page", [1, 16, 48, 128])
@pytest.mark.parametrize("B,hi", [(1, 1), (1, 5000), (3, 40), (64, 2), (700, 30), (1024, 3),
                                  (1025, 2), (4096, 9)])
def test_page_tables(cuda, B, hi, page):
    rng = random.Random(B * 13 + hi)
    cached = [rng.randint(0, 200) for _ in range(B)]
    new = [rng.randint(0, hi) for _ in range(B)]
    cached[0], new[-1] = 0, hi
    _tables_case(cuda, cached, new, page, -(-(200 + hi) // page))


def test_page_tables_edges(cuda):
    _tables_case(cuda, [], [], 16, 4)
    _tables_case(cuda, [0, 0], [0, 0], 16, 4)
    _tables_case(cuda, [16, 15, 17, 0], [1, 1, 1, 16], 16, 4, pad=0)
    _tables_case(cuda, [16, 15, 17, 0], [1, 1, 1, 16], 16, 4, pad=5000)  # several blocks
    _tables_case(cuda, [5, 3, 64], [70, 1, 2], 16, 9, in_place=True, stride=3)
    _tables_case(cuda, [5] * 900, [7] * 900, 16, 9, in_place=True)
    # the stack runs dry: the second request and the last one get nothing, the third needs nothing
    _tables_case(cuda, [16, 16, 3, 16], [16, 32, 4, 1], 16, 8, count=2)
    _tables_case(cuda, [0, 0], [16, 16], 16, 8, count=0)
    # a full row
    _tables_case(cuda, [30, 2], [5, 5], 16, 2)


def test_page_tables_bad_lengths_are_recorded(cuda):
    def ints(v, dtype=torch.int32):
        return torch.tensor(v, dtype=dtype, device=cuda)

    for cached, new in (([-1, 3], [2, 2]), ([9999, 3], [2, 2]), ([1, 3], [-2, 2]), ([1, 3], [2**31 - 1, 2])):
        seq, cu, pos, slots = ints([0, 0]), ints([0] * 3), ints([0] * 8), ints([0] * 8, torch.int64)
        tables, err = ints([[0, -1], [1, -1]]), ints([0])
        ops.build_page_tables(ints(cached), ints(new), 16, tables, ints([2, 3]), ints([2]),
                              seq_lens=seq, cu_q=cu, positions=pos, slot_mapping=slots,
                              free_count_out=ints([0]), err_word=err)
        assert err.item() == 6
        assert 0 <= cu[1] <= cu[2] <= 8 and seq.tolist()[1] == 5
        assert tables.tolist() == [[0, -1], [1, -1]]
    # more tokens than the step's buffers hold: cut, nothing past them written
    pos, slots, cu, err = ints([0] * 4), ints([0] * 4, torch.int64), ints([0] * 3), ints([0])
    ops.build_page_tables(ints([0, 0]), ints([3, 3]), 16, ints([[-1], [-1]]), ints([0, 1]), ints([2]),
                          seq_lens=ints([0, 0]), cu_q=cu, positions=pos, slot_mapping=slots,
                          err_word=err)
    assert err.item() == 6 and cu.tolist() == [0, 3, 4] and pos.tolist() == [0, 1, 2, 0]


def test_release_pages_and_reuse(cuda):
    def ints(v, dtype=torch.int32):
        return torch.tensor(v, dtype=dtype, device=cuda)

    tables = ints([[4, 5, -1], [6, -1, -1], [7, 8, 9]])
    lens, free, count, err = ints([20, 16, 48]), ints([0, 1, -1, -1, -1, -1, -1, -1]), ints([2]), ints([0])
    ops.release_pages(ints([2, 0, 2]), lens, 16, tables, free, count, err)
    assert free.tolist() == [0, 1, 7, 8, 9, 4, 5, -1] and count.item() == 7
    assert lens.tolist() == [0, 16, 0] and tables.tolist() == [[-1] * 3, [6, -1, -1], [-1] * 3]
    assert err.item() == 0
    ops.release_pages(ints([5]), lens, 16, tables, free, count, err)
    assert err.item() == 6 and count.item() == 7


# ------------------------------------------------------------------------ rope + cache write
def _rope64(x, w, cs, R, interleaved, eps):
    """x [T, heads, D] in 64 bits: (value, magnitude of the terms)."""
    z = x.double()
    if w is not None:
        z = z / ((z * z).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    c, s = cs[:, None, :R // 2].double(), cs[:, None, R // 2:].double()
    i = torch.arange(R // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    out, mag = z.clone(), z.abs()
    out[..., a], out[..., b] = z[..., a] * c - z[..., b] * s, z[..., b] * c + z[..., a] * s
    mag[..., a] = mag[..., b] = z[..., a].abs() + z[..., b].abs()
    return out, mag


@pytest.mark.parametrize("T,Hq,Hkv,D,R,page,inter,norm,layout", [
    (1, 1, 1, 64, 64, 16, False, False, "split"),
    (16, 32, 4, 128, 128, 16, False, True, "split"),
    (16, 32, 4, 128, 128, 16, True, True, "joint"),
    (513, 14, 2, 64, 32, 48, False, False, "joint"),
    (77, 5, 1, 128, 64, 128, True, False, "heads"),
    (300, 8, 8, 128, 2, 32, False, True, "heads"),
    (33, 7, 1, 64, 0, 16, False, True, "split"),
    (33, 6, 2, 64, 30, 16, True, True, "split"),
    (33, 6, 2, 128, 6, 16, False, False, "split"),
    (2100, 12, 4, 128, 128, 64, False, True, "split")])
def test_rope_cache_write(cuda, T, Hq, Hkv, D, R, page, inter, norm, layout):
    g = _gen(cuda, T + Hq * 3 + D)
    pages = -(-T // page) + 3
    cache = {"split": lambda: [_bf16(g, pages, page, Hkv, D) for _ in range(2)],
             "joint": lambda: list(_bf16(g, pages, 2, page, Hkv, D).unbind(1)),
             "heads": lambda: [_bf16(g, pages, Hkv, page, D).transpose(1, 2) for _ in range(2)]}[layout]
    kc, vc = cache()
    qkv = _bf16(g, T, (Hq + 2 * Hkv) * D + 16, std=2.0)[:, :(Hq + 2 * Hkv) * D]
    angle = torch.rand(4096, max(R // 2, 1), device=cuda, generator=g, dtype=torch.float64) * 50
    cs = torch.cat([angle.cos(), angle.sin()], 1).float()[:, :R].contiguous()
    pos = torch.randint(4096, (T,), device=cuda, generator=g, dtype=torch.int32)
    slots = torch.randperm(pages * page, device=cuda, generator=g)[:T].clone()
    if T > 2:
        slots[T // 2] = -1
    qw, kw = (_bf16(g, D), _bf16(g, D)) if norm else (None, None)
    q = torch.empty(T, Hq, D, dtype=torch.bfloat16, device=cuda)
    want_k, want_v = kc.double(), vc.double()
    x = qkv.reshape(T, Hq + 2 * Hkv, D)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    ops.rope_cache_write(qkv, pos, slots, cs, kc, vc, q, q_norm_weight=qw, k_norm_weight=kw,
                         eps=1e-6, interleaved=inter, err_word=err)
    qd, qm = _rope64(x[:, :Hq], qw, cs[pos.long()], R, inter, 1e-6)
    kd, km = _rope64(x[:, Hq:Hq + Hkv], kw, cs[pos.long()], R, inter, 1e-6)
    _within(q, qd, BF16 * qd.abs() + SUMS * qm)
    live = slots >= 0
    at = (slots[live] // page, slots[live] % page)
    bound = torch.zeros_like(want_k)
    want_k[at], bound[at] = kd[live], (BF16 * kd.abs() + SUMS * km)[live]
    want_v[at] = x[:, Hq + Hkv:].double()[live]
    _within(kc, want_k, bound)  # everything else as it was
    assert torch.equal(vc.double(), want_v) and err.item() == 0
    # q over its own part of qkv gives the same values
    kc2, vc2 = cache()
    ops.rope_cache_write(qkv, pos, slots, cs, kc2, vc2, qkv[:, :Hq * D].unflatten(1, (Hq, D)),
                         q_norm_weight=qw, k_norm_weight=kw, eps=1e-6, interleaved=inter)
    assert torch.equal(qkv[:, :Hq * D].reshape(T, Hq, D), q)


def test_rope_out_of_range_is_recorded(cuda):
    g = _gen(cuda, 1)
    kc, vc = _bf16(g, 2, 16, 1, 64), _bf16(g, 2, 16, 1, 64)
    kept = kc.clone()
    cs = torch.ones(8, 64, device=cuda)
    q = torch.empty(1, 2, 64, dtype=torch.bfloat16, device=cuda)
    for pos, slot, code in ((0, 32, 7), (0, 2**40, 7), (8, -1, 8), (-1, -1, 8)):
        err = torch.zeros(1, dtype=torch.int32, device=cuda)
        ops.rope_cache_write(_bf16(g, 1, 256), torch.tensor([pos], dtype=torch.int32, device=cuda),
                             torch.tensor([slot], device=cuda), cs, kc, vc, q, err_word=err)
        assert err.item() == code and torch.equal(kc, kept)


# -------------------------------------------------------------------------------- attention
def _attention64(q, kc, vc, tables, seq, cu, scale, window):
    T, Hq, D = q.shape
    page, Hkv = kc.shape[1], kc.shape[2]
    out = torch.full((T, Hq, D), math.nan, dtype=torch.float64, device=q.device)
    lse = torch.full((T, Hq), math.nan, dtype=torch.float64, device=q.device)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(len(seq)):
        n, L = cu[b + 1] - cu[b], seq[b]
        ids = tables[b][:-(-L // page)].long().clamp(min=0)
        k = kc[ids].reshape(-1, Hkv, D)[:L].double()
        v = vc[ids].reshape(-1, Hkv, D)[:L].double()
        p = (L - n + torch.arange(n, device=q.device))[:, None]
        j = torch.arange(L, device=q.device)[None, :]
        seen = (j <= p) & (j > p - window if window else True)
        for h in range(Hq):
            qd = q[cu[b]:cu[b + 1], h].double()
            kh, vh = k[:, h * Hkv // Hq], v[:, h * Hkv // Hq]
            used = seen.any(0)  # keys that no row sees may hold anything
            kh, vh = torch.where(used[:, None], kh, 0.0), torch.where(used[:, None], vh, 0.0)
            z = (qd @ kh.t() * scale).masked_fill(~seen, -math.inf)
            top = z.amax(1, keepdim=True) if L else torch.full((n, 1), -math.inf, device=q.device)
            w = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
            total = w.sum(1, keepdim=True)
            w = w / torch.where(total == 0, 1.0, total)
            o, mag = w @ vh, w @ vh.abs()
            out[cu[b]:cu[b + 1], h] = o
            lse[cu[b]:cu[b + 1], h] = (top + total.log())[:, 0]
            err = D * 2.0 ** -24 * scale * ((qd.abs() @ kh.abs().t()) * seen).amax(1) if L else torch.zeros(n, device=q.device)
            # a score error of e moves every weight by at most 2 e
            tol[cu[b]:cu[b + 1], h] = BF16 * (o.abs() + mag) * 1.01 + (SUMS + 2 * err[:, None]) * mag
            ltol[cu[b]:cu[b + 1], h] = err + 2.0 ** -20 * (1 + lse[cu[b]:cu[b + 1], h].nan_to_num(neginf=0.0).abs())
    return out, lse, tol, ltol


def _attention_case(cuda, lens, Hq, Hkv, D, page, window=0, layout="split", seed=0, stale=math.nan,
                    max_q=None, spread=1.0, workspace=None, scale=None):
    """lens: (sequence length, new tokens) per request."""
    g = _gen(cuda, seed + Hq * 7 + D + page + len(lens))
    seq, new = [s for s, _ in lens], [n for _, n in lens]
    held = [-(-s // page) for s in seq]
    pages = sum(held) + 2
    ids = torch.randperm(pages, device=cuda, generator=g, dtype=torch.int32)
    tables = torch.full((len(lens), max(held + [1]) + 1), -1, dtype=torch.int32, device=cuda)
    cu, at = [0], 0
    for b, n in enumerate(new):
        tables[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
        cu.append(cu[-1] + n)
    kc, vc = {"split": lambda: [_bf16(g, pages, page, Hkv, D) for _ in range(2)],
              "joint": lambda: list(_bf16(g, pages, 2, page, Hkv, D).unbind(1)),
              "heads": lambda: [_bf16(g, pages, Hkv, page, D).transpose(1, 2) for _ in range(2)]}[layout]()
    # what the cache holds past a sequence, in unused pages and out of every window is stale
    alive = torch.zeros(pages, page, dtype=torch.bool, device=cuda)
    for b, (s, n) in enumerate(lens):
        first = max(0, s - n - window + 1) if window else 0
        j = torch.arange(min(first, s), s, device=cuda)
        alive[tables[b, j // page].long(), j % page] = True
        if window:
            tables[b, :first // page] = -1  # pages that left the window were given back
    kc[~alive] = stale
    vc[~alive] = stale
    T = cu[-1]
    q = _bf16(g, T, Hq + 1, D, std=spread)[:, :Hq]
    out = torch.full((T, Hq, D + 8), 7.0, dtype=torch.bfloat16, device=cuda)[..., :D]
    lse = torch.empty(T, Hq, device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    ws = ops.attention_workspace(cuda) if workspace is None else workspace
    scale_ = D ** -0.5 if scale is None else scale

    def call():
        ops.paged_attention(q, kc, vc, tables, torch.tensor(seq, dtype=torch.int32, device=cuda),
                            torch.tensor(cu, dtype=torch.int32, device=cuda), out,
                            max_q_len=max(new + [0]) if max_q is None else max_q, workspace=ws,
                            window=window, lse=lse, err_word=err, scale=scale)

    call()
    want, wlse, tol, ltol = _attention64(q, kc, vc, tables, seq, cu, scale_, window)
    assert err.item() == 0
    _within(out, want, tol)
    empty = wlse == -math.inf
    assert torch.equal(lse == -math.inf, empty) and (out[empty] == 0).all()
    _within(lse[~empty], wlse[~empty], ltol[~empty])
    first = out.clone(), lse.clone()
    call()  # the same bits again, with the workspace as the first call left it
    assert torch.equal(out, first[0]) and torch.equal(lse, first[1])
    return out, ws


@pytest.mark.parametrize("Hq,Hkv,D,page", [(1, 1, 64, 16), (32, 4, 128, 16), (14, 2, 64, 48),
                                           (5, 1, 128, 32), (8, 8, 128, 128), (64, 4, 128, 64),
                                           (32, 1, 64, 16), (36, 2, 128, 16)])
@pytest.mark.parametrize("lens", [
    [(1, 1)], [(17, 1)], [(0, 1)], [(3000, 1)], [(1280, 1), (1, 1), (129, 1), (128, 1), (0, 0)],
    [(5, 5)], [(130, 130)], [(700, 33), (1, 1), (257, 257), (64, 0), (300, 2)], [(2, 6), (0, 3)],
    [(1000, 300)]], ids=str)
def test_attention(cuda, Hq, Hkv, D, page, lens):
    _attention_case(cuda, lens, Hq, Hkv, D, page)


@pytest.mark.parametrize("window", [1, 16, 100, 129, 5000])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 1, 128), (4, 4, 64), (64, 4, 64)])
def test_attention_window(cuda, Hq, Hkv, D, window):
    _attention_case(cuda, [(700, 1), (513, 200), (90, 90), (1, 1), (400, 16)], Hq, Hkv, D, 16, window=window)


@pytest.mark.parametrize("layout", ["joint", "heads"])
@pytest.mark.parametrize("stale", [math.nan, math.inf, -math.inf, 3e38])
def test_attention_cache_layouts_and_stale_pages(cuda, layout, stale):
    _attention_case(cuda, [(333, 1), (150, 150), (1000, 77)], 16, 2, 128, 32, layout=layout, stale=stale)


@pytest.mark.parametrize("spread", [0.0, 30.0])
def test_attention_flat_and_peaked(cuda, spread):
    _attention_case(cuda, [(2000, 1), (600, 300)], 8, 2, 128, 16, spread=spread)
    _attention_case(cuda, [(2000, 1), (600, 300)], 8, 2, 128, 16, spread=1.0, scale=0.0)


def test_attention_long_sequences_and_many_requests(cuda):
    _, ws = _attention_case(cuda, [(70001, 1)], 4, 1, 128, 64)
    _attention_case(cuda, [(40000, 40)], 8, 1, 64, 16, workspace=ws)
    rng = random.Random(3)
    _attention_case(cuda, [(rng.randint(1, 90), 1) for _ in range(1500)], 2, 1, 64, 16, workspace=ws)
    _attention_case(cuda, [(rng.randint(40, 90), rng.randint(0, 40)) for _ in range(300)], 6, 2, 64, 16,
                    workspace=ws)


@pytest.mark.parametrize("max_q", [0, 1, 100000])
def test_attention_hint_only_chooses_kernels(cuda, max_q):
    _attention_case(cuda, [(300, 1), (500, 200), (64, 3)], 8, 2, 128, 16, max_q=max_q)


def test_attention_offsets_past_32_bits(cuda):
    """Pages of a cache with more than 2^32 bytes between them."""
    page, Hkv, D, far = 16, 2, 128, 600_000
    kc = torch.empty(far + 4, page, Hkv, D, dtype=torch.bfloat16, device=cuda)
    vc = torch.empty_like(kc)
    assert kc[0].numel() * far > 2 ** 31
    g = _gen(cuda, 5)
    ids = torch.tensor([[far + 3, 1, far, 7]], dtype=torch.int32, device=cuda)
    for c in (kc, vc):
        c[ids[0].long()] = _bf16(g, 4, page, Hkv, D)
    ws = ops.attention_workspace(cuda)
    for n in (1, 50):
        q = _bf16(g, n, 8, D)
        out = torch.empty_like(q)
        ops.paged_attention(q, kc, vc, ids, torch.tensor([60], dtype=torch.int32, device=cuda),
                            torch.tensor([0, n], dtype=torch.int32, device=cuda), out, max_q_len=n, workspace=ws)
        want, _, tol, _ = _attention64(q, kc, vc, ids, [60], [0, n], D ** -0.5, 0)
        _within(out, want, tol)
    slots = torch.tensor([(far + 2) * page + 5], device=cuda)
    qkv = _bf16(g, 1, 12 * D)
    ops.rope_cache_write(qkv, torch.zeros(1, dtype=torch.int32, device=cuda), slots,
                         torch.cat([torch.ones(1, 64, device=cuda), torch.zeros(1, 64, device=cuda)], 1),
                         kc, vc, torch.empty(1, 8, D, dtype=torch.bfloat16, device=cuda))
    assert torch.equal(kc[far + 2, 5], qkv.view(12, D)[8:10]) and torch.equal(vc[far + 2, 5], qkv.view(12, D)[10:])


def test_attention_bad_inputs_are_recorded_not_read(cuda):
    g = _gen(cuda, 2)
    kc, vc, q = _bf16(g, 4, 16, 1, 64), _bf16(g, 4, 16, 1, 64), _bf16(g, 4, 2, 64)
    ws = ops.attention_workspace(cuda)

    def run(tables, seq, cu, max_q):
        out = torch.full_like(q, 7.0)
        err = torch.zeros(1, dtype=torch.int32, device=cuda)
        ints = [torch.tensor(v, dtype=torch.int32, device=cuda) for v in (tables, seq, cu)]
        ops.paged_attention(q, kc, vc, *ints, out, max_q_len=max_q, workspace=ws, err_word=err)
        return out, err.item()

    for max_q in (1, 64):
        assert run([[4, 0]], [20], [0, 4], max_q)[1] == 7
        assert run([[0, -1]], [20], [0, 4], max_q)[1] == 7
        assert run([[0, 1]], [33], [0, 4], max_q)[1] == 6
        assert run([[0, 1]], [-3], [0, 4], max_q)[1] == 6
        out, err = run([[0, 1]], [20], [0, 5], max_q)
        assert err == 6 and (out == 7.0).all()
        assert run([[0, 1]], [20], [3, 1], max_q)[1] == 6
        # tokens of no request stay as they were
        out, err = run([[0, 1]], [20], [1, 3], max_q)
        assert err == 0 and (out[0] == 7.0).all() and (out[3] == 7.0).all() and (out[1:3] != 7.0).all()


def test_operators_replay_from_a_graph_with_new_lengths(cuda):
    """One captured step serves other lengths: everything that changes is read on the device."""
    B, page, Hq, Hkv, D = 5, 16, 8, 2, 128
    g = _gen(cuda, 11)
    i32 = dict(dtype=torch.int32, device=cuda)
    kc, vc = _bf16(g, 64, page, Hkv, D), _bf16(g, 64, page, Hkv, D)
    tables, free = torch.full((B, 12), -1, **i32), torch.arange(64, **i32)
    count, lens, new = torch.tensor([64], **i32), torch.zeros(B, **i32), torch.zeros(B, **i32)
    seq, cu, pos = torch.zeros(B, **i32), torch.zeros(B + 1, **i32), torch.zeros(40, **i32)
    slots, err = torch.zeros(40, dtype=torch.int64, device=cuda), torch.zeros(1, **i32)
    qkv = torch.zeros(40, (Hq + 2 * Hkv) * D, dtype=torch.bfloat16, device=cuda)
    q, out = (torch.zeros(40, Hq, D, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    cs = torch.cat([torch.ones(256, 64, device=cuda), torch.zeros(256, 64, device=cuda)], 1)
    ws = ops.attention_workspace(cuda)

    def step():
        ops.build_page_tables(lens, new, page, tables, free, count, seq_lens=seq, cu_q=cu,
                              positions=pos, slot_mapping=slots, err_word=err)
        ops.rope_cache_write(qkv, pos, slots, cs, kc, vc, q, err_word=err)
        ops.paged_attention(q, kc, vc, tables, seq, cu, out, max_q_len=40, workspace=ws, err_word=err)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    had = [0] * B
    for n in ([7, 0, 20, 1, 3], [1, 1, 1, 0, 1], [0, 30, 1, 1, 2], [1, 1, 1, 1, 1]):
        lens.copy_(torch.tensor(had, **i32))
        new.copy_(torch.tensor(n, **i32))
        qkv.copy_(_bf16(g, *qkv.shape))
        graph.replay()
        had = [a + b for a, b in zip(had, n)]
        cl = [0]
        for v in n:
            cl.append(cl[-1] + v)
        assert seq.tolist() == had and cu.tolist() == cl and err.item() == 0
        assert count.item() == 64 - sum(-(-h // page) for h in had)
        T = cl[-1]
        want, _, tol, _ = _attention64(qkv[:T, :Hq * D].reshape(T, Hq, D), kc, vc, tables, had, cl, D ** -0.5, 0)
        _within(out[:T], want, tol)
        x = qkv[:T].view(T, Hq + 2 * Hkv, D)
        s = slots[:T]
        assert torch.equal(kc[s // page, s % page], x[:, Hq:Hq + Hkv])
        assert (slots[T:] == -1).all()


def test_operators_on_another_stream(cuda):
    g = _gen(cuda, 4)
    x, w = _bf16(g, 64, 2048), _bf16(g, 2048)
    a, b = torch.empty_like(x), torch.empty_like(x)
    ops.add_rms_norm(x, w, out=a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        y = x * 1  # queued behind the sleep: a launch elsewhere would read it too early
        ops.add_rms_norm(y, w, out=b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b)


# --------------------------------------------------------------------------------- refusals
def test_refusals(cuda):
    g = _gen(cuda, 9)
    x, w = _bf16(g, 4, 64), _bf16(g, 64)
    out = torch.empty_like(x)
    f8, sc = torch.empty(4, 64, dtype=torch.float8_e4m3fn, device=cuda), torch.empty(4, 1, device=cuda)
    for kw in (dict(), dict(out=out, out_fp8=f8, scales=sc), dict(out=out.float()), dict(out=out[:3]),
               dict(out=out.cpu()), dict(out_fp8=f8), dict(out_fp8=f8, scales=sc, group_size=48),
               dict(out_fp8=f8, scales=sc, group_size=32), dict(out=out, scales=sc),
               dict(out=out, residual=x[:, :32]), dict(out=out.t().contiguous().t())):
        with pytest.raises(ValueError):
            ops.add_rms_norm(x, w, **kw)
    with pytest.raises(ValueError):
        ops.add_rms_norm(x[:1].expand(4, 64), w, out=out[:1].expand(4, 64))
    with pytest.raises(RuntimeError, match="16384"):
        big = torch.zeros(1, 16385, dtype=torch.bfloat16, device=cuda)
        ops.add_rms_norm(big, big[0], out=torch.empty_like(big))

    i32 = dict(dtype=torch.int32, device=cuda)
    kc = _bf16(g, 4, 16, 2, 64)
    q, ws = _bf16(g, 2, 4, 64), ops.attention_workspace(cuda)
    args = dict(q=q, k_cache=kc, v_cache=kc, block_tables=torch.zeros(1, 4, **i32),
                seq_lens=torch.tensor([2], **i32), cu_q=torch.tensor([0, 2], **i32), out=torch.empty_like(q))
    for change in (dict(q=q.float()), dict(out=q[:1]), dict(k_cache=kc[0]), dict(v_cache=kc[:, :8]),
                   dict(cu_q=torch.zeros(3, **i32)), dict(seq_lens=torch.zeros(1, device=cuda)),
                   dict(block_tables=torch.zeros(1, 4, dtype=torch.int64, device=cuda)),
                   dict(q=_bf16(g, 2, 64, 4).transpose(1, 2))):
        with pytest.raises(ValueError):
            ops.paged_attention(**{**args, **change}, max_q_len=2, workspace=ws)
    for change, kw in ((dict(q=q[:, :3], out=torch.empty_like(q[:, :3])), {}), ({}, dict(workspace=ws[:64])),
                       ({}, dict(window=-1)), ({}, dict(max_q_len=-1)),
                       (dict(k_cache=_bf16(g, 4, 8, 2, 64), v_cache=_bf16(g, 4, 8, 2, 64)), {}),
                       (dict(q=_bf16(g, 2, 4, 68)[..., 2:66]), {})):
        with pytest.raises(RuntimeError, match="lm_paged_attention"):
            ops.paged_attention(**{**args, **change}, **{**dict(max_q_len=2, workspace=ws), **kw})
    k96 = _bf16(g, 4, 16, 2, 96)
    q96 = _bf16(g, 2, 4, 96)
    with pytest.raises(RuntimeError, match="head_dim"):
        ops.paged_attention(**{**args, "q": q96, "out": q96, "k_cache": k96, "v_cache": k96}, max_q_len=2,
                            workspace=ws)

    rope = dict(qkv=_bf16(g, 2, 8 * 64), positions=torch.zeros(2, **i32),
                slot_mapping=torch.zeros(2, dtype=torch.int64, device=cuda), cos_sin=torch.ones(4, 64, device=cuda),
                k_cache=kc, v_cache=kc.clone(), q_out=torch.empty_like(q))
    for change in (dict(qkv=_bf16(g, 2, 7 * 64)), dict(slot_mapping=torch.zeros(2, **i32)),
                   dict(cos_sin=torch.ones(4, 64, device=cuda).bfloat16()), dict(positions=torch.zeros(3, **i32))):
        with pytest.raises(ValueError):
            ops.rope_cache_write(**{**rope, **change})
    for change in (dict(cos_sin=torch.ones(4, 66, device=cuda)), dict(cos_sin=torch.ones(4, 33, device=cuda))):
        with pytest.raises(RuntimeError, match="rot_dim"):
            ops.rope_cache_write(**{**rope, **change})

    tab = dict(cached_lens=torch.zeros(2, **i32), new_lens=torch.ones(2, **i32), page_size=16,
               block_tables=torch.full((2, 2), -1, **i32), free_pages=torch.arange(4, **i32),
               free_count=torch.tensor([4], **i32), seq_lens=torch.zeros(2, **i32), cu_q=torch.zeros(3, **i32),
               positions=torch.zeros(2, **i32), slot_mapping=torch.zeros(2, dtype=torch.int64, device=cuda))
    for change in (dict(cu_q=torch.zeros(2, **i32)), dict(slot_mapping=torch.zeros(2, **i32)),
                   dict(new_lens=torch.ones(3, **i32)), dict(block_tables=torch.zeros(2, 0, **i32))):
        with pytest.raises(ValueError):
            ops.build_page_tables(**{**tab, **change})
    with pytest.raises(RuntimeError, match="sizes"):
        ops.build_page_tables(**{**tab, "page_size": 0})
    with pytest.raises(RuntimeError, match="4096"):
        many = torch.zeros(4097, **i32)
        ops.build_page_tables(**{**tab, "cached_lens": many, "new_lens": many, "seq_lens": many,
                                 "cu_q": torch.zeros(4098, **i32), "block_tables": torch.zeros(4097, 1, **i32)})
    assert _lib.DEVERR_NAMES[5]


@pytest.mark.parametrize("T,Hq,Hkv,D,R,inter,norm", [(2049, 40, 8, 64, 64, False, True),
                                                     (2048, 33, 11, 128, 64, True, False),
                                                     (2500, 9, 3, 128, 128, False, False)])
def test_rope_cache_write_of_many_tokens(cuda, T, Hq, Hkv, D, R, inter, norm):
    """Sizes at which a warp takes several groups of query heads, the last of them ragged."""
    test_rope_cache_write(cuda, T, Hq, Hkv, D, R, 16, inter, norm, "split")


@pytest.mark.parametrize("D", [64, 128])
def test_attention_negative_scale(cuda, D):
    """A scale's sign may stand in the queries: the same bits."""
    g = _gen(cuda, D)
    kc, vc = _bf16(g, 40, 16, 2, D), _bf16(g, 40, 16, 2, D)
    tables = torch.randperm(40, device=cuda, generator=g).to(torch.int32).view(2, 20)
    ws = ops.attention_workspace(cuda)
    for new in ([1, 1], [300, 70]):
        cu = torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device=cuda)
        seq = torch.tensor([310, 150], dtype=torch.int32, device=cuda)
        q = _bf16(g, sum(new), 8, D)
        outs = []
        for sign in (1, -1):
            out, lse = torch.empty_like(q), torch.empty(sum(new), 8, device=cuda)
            ops.paged_attention(q * sign, kc, vc, tables, seq, cu, out, max_q_len=max(new), workspace=ws,
                                scale=0.15 * sign, lse=lse)
            outs.append((out, lse))
        assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def test_attention_k_and_v_of_different_layouts(cuda):
    """K with tokens before heads and V with heads before tokens, one kv head, one page, strides of one-sized
    dimensions that mean nothing."""
    g = _gen(cuda, 21)
    ws = ops.attention_workspace(cuda)
    for pages, Hkv in ((9, 2), (9, 1), (1, 2), (1, 1)):
        kc = _bf16(g, pages, 16, Hkv, 64)
        vc = _bf16(g, pages, Hkv, 16, 64).transpose(1, 2)
        if Hkv == 1:
            kc = kc.as_strided(kc.shape, (kc.stride(0), kc.stride(1), 0, 1))
        if pages == 1:
            vc = vc.as_strided(vc.shape, (0, *vc.stride()[1:]))
        L = pages * 16 - 3
        tables = torch.randperm(pages, device=cuda, generator=g).to(torch.int32)[None]
        for n in (1, min(L, 50)):
            q = _bf16(g, n, 4 * Hkv, 64)
            out = torch.empty_like(q)
            ops.paged_attention(q, kc, vc, tables, torch.tensor([L], dtype=torch.int32, device=cuda),
                                torch.tensor([0, n], dtype=torch.int32, device=cuda), out, max_q_len=n,
                                workspace=ws)
            want, _, tol, _ = _attention64(q, kc, vc, tables, [L], [0, n], 64 ** -0.5, 0)
            _within(out, want, tol)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("B", [2, 13, 70, 149, 600])
def test_attention_work_cut_anywhere(cuda, B, new):
    """Lengths that let the CTAs' equal shares begin and end at every place of an item: ahead of its first block,
    between its blocks, behind its last."""
    rng = random.Random(B + new)
    ws = ops.attention_workspace(cuda)
    for top in (130, 700, 3000 if B < 100 else 1300):
        _attention_case(cuda, [(rng.randint(0, top), rng.randint(1, new)) for _ in range(B)], 8, 1, 64, 16,
                        workspace=ws, seed=top)


def _keyless_runs(rng, B, run, top):
    """Single tokens over 1 .. top keys, with runs of requests without any at the front, in the middle and
    at the end, and further runs of other lengths between them."""
    lens = [(rng.randint(1, top), 1) for _ in range(B)]
    for at in (0, B // 2, B - run, B // 5, B // 3 + 1):
        lens[at:at + run] = [(0, 1)] * run
    for at in range(B // 2 + 20, B - 20, 11):
        n = rng.randint(1, 9)
        lens[at:at + n] = [(0, 1)] * n
    return lens


@pytest.mark.parametrize("run", [1, 2, 9])
@pytest.mark.parametrize("Hkv", [8, 4, 2, 1])
def test_attention_requests_without_keys_among_others(cuda, Hkv, run):
    """Padded rows of a decode batch: their segments take no turn of the query ring."""
    rng = random.Random(Hkv * 10 + run)
    _, ws = _attention_case(cuda, _keyless_runs(rng, 512, run, 500), 2 * Hkv, Hkv, 64, 16)
    one = [(500, 1)] * 512
    one[:run] = [(0, 1)] * run
    _attention_case(cuda, one, Hkv, Hkv, 64, 16, workspace=ws)


def test_attention_requests_without_keys_in_long_and_mixed_batches(cuda):
    rng = random.Random(1)
    _, ws = _attention_case(cuda, _keyless_runs(rng, 3000, 4, 60), 4, 2, 128, 16)
    _attention_case(cuda, _keyless_runs(rng, 600, 3, 2500), 4, 4, 64, 64, workspace=ws)
    # beside the tensor-core kernel, whose own requests have some without keys, too
    lens = _keyless_runs(rng, 400, 3, 700) + [(700, 200), (0, 50), (3, 90), (0, 200)]
    rng.shuffle(lens)
    _attention_case(cuda, lens, 8, 4, 64, 16, workspace=ws)


def test_page_tables_of_any_number_of_requests(cuda):
    """Counts around the one whose shared memory, static part included, passes 48 KB: in a process of
    their own, since a larger call before them would have raised the kernel's limit."""
    code = ("import torch, tests.test_gpu_decoder_ops as t\n"
            "for B in (4052, 4053, 4054, 4095, 4096):\n"
            "    t._tables_case(torch.device('cuda', 0), [3] * B, [1] * (B - 1) + [40], 16, 4)\n")
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("cached,new,T,page", [
    ([5, 0, 30], [20, 24, 3], 25, 16),  # the second request keeps 5 tokens, the third none
    ([0, 0, 0], [40, 40, 9], 42, 16),  # the second request's first page, none for the third
    ([0, 0], [40, 40], 0, 16),
    ([16] * 1100, [9] * 1100, 5003, 16),  # several blocks
    ([7] * 4096, [3] * 4096, 6001, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_page_tables_cut_tokens_hold_no_pages(cuda, cached, new, T, page, in_place):
    """A step with more tokens than its buffers hold gives what the step of the tokens that fit would give."""
    B, room, kept = len(cached), T, []
    for n in new:
        kept.append(min(n, room))
        room -= kept[-1]
    width = max(1, -(-max(c + n for c, n in zip(cached, kept)) // page))  # too narrow for some of the cut rows
    have = [-(-c // page) for c in cached]
    grants = sum(-(-(c + n) // page) - h for c, n, h in zip(cached, kept, have))
    pool = list(range(sum(have) + grants))  # and no page more than the kept tokens need
    random.Random(T).shuffle(pool)
    tables, at = [[-1] * width for _ in range(B)], 0
    for b, h in enumerate(have):
        tables[b][:h] = pool[at:at + h]
        at += h
    free = pool[at:]

    def ints(v, dtype=torch.int32):
        return torch.tensor(v, dtype=dtype, device=cuda)

    dt, lens, dfree, count, err = ints(tables), ints(cached), ints(free + [-7]), ints([len(free)]), ints([0])
    seq = lens if in_place else ints([-5] * B)
    left = count if in_place else ints([-5])
    cu, pos, slots = ints([-5] * (B + 1)), ints([-5] * T), ints([-5] * T, torch.int64)
    ops.build_page_tables(lens, ints(new), page, dt, dfree, count, seq_lens=seq, cu_q=cu, positions=pos,
                          slot_mapping=slots, free_count_out=left, err_word=err)
    want = _tables_by_hand(cached, kept, page, tables, free, len(free), T)
    assert (seq.tolist(), cu.tolist(), pos.tolist(), slots.tolist(), left.item()) == want[:5]
    assert dt.tolist() == tables and err.item() == 6
    if in_place:  # every page comes back
        ops.release_pages(torch.arange(B, dtype=torch.int32, device=cuda), lens, page, dt,
                          (every := ints([-1] * (len(pool) + 1))), (n := ints([0])))
        assert n.item() == len(pool) - left.item() == sum(have) + grants
        assert sorted(every.tolist()) == sorted(pool + [-1])


def test_release_pages_passes_over_entries_without_a_page(cuda):
    """Pages that left a window were given back already: their entries are negative."""
    def ints(v, dtype=torch.int32):
        return torch.tensor(v, dtype=dtype, device=cuda)

    tables, lens = ints([[-1, -1, 7], [4, 5, -1], [-1, 9, -1]]), ints([48, 20, 33])
    free, count, err = ints([0, -8, -8, -8, -8]), ints([1]), ints([0])
    ops.release_pages(ints([0, 2, 1]), lens, 16, tables, free, count, err)
    assert free.tolist() == [0, 7, 9, 4, 5] and count.item() == 5 and err.item() == 0
    assert lens.tolist() == [0, 0, 0] and tables.tolist() == [[-1] * 3] * 3
    # long rows, more entries than the stack has room for and just as many pages
    rng = random.Random(4)
    rows = [[rng.choice([-1, -1, b * 1000 + i]) for i in range(700)] for b in range(3)]
    want = [i for b in (2, 0, 1) for i in rows[b][:620] if i >= 0]
    tables, lens = ints(rows), ints([620] * 3)
    free, count = ints([-8] * (len(want) + 1)), ints([0])
    ops.release_pages(ints([2, 0, 1]), lens, 1, tables, free, count, err)
    assert free.tolist() == want + [-8] and count.item() == len(want) and err.item() == 0
    assert tables.tolist() == [[-1] * 620 + r[620:] for r in rows]
    # a page too many: the row stays as it is, the others go back
    tables, lens = ints([[1, -1, 2], [3, 4, 5]]), ints([3, 3])
    free, count = ints([-8] * 4), ints([0])
    ops.release_pages(ints([0, 1]), lens, 1, tables, free, count, err)
    assert free.tolist() == [1, 2, -8, -8] and count.item() == 2 and err.item() == 6
    assert lens.tolist() == [0, 3] and tables.tolist() == [[-1] * 3, [3, 4, 5]]


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 2 ** 30])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 1, 128), (2, 2, 64)])
def test_attention_window_past_every_key(cuda, Hq, Hkv, D, window):
    """Windows that stand for none, also where the first queries come before every key; both kernels."""
    for max_q in (1, 1000):
        _attention_case(cuda, [(2, 6), (5, 5), (0, 3), (1, 1), (300, 1)], Hq, Hkv, D, 16, window=window,
                        max_q=max_q)
    _attention_case(cuda, [(2, 6), (150, 400), (300, 300), (0, 300), (700, 1)], Hq, Hkv, D, 16, window=window)


@pytest.mark.parametrize("B,T,page,hint", [
    (4096, 1024, 1024, 1024), (4096, 1024, 1024, 1), (32, 20480, 4096, 20480), (32, 16384, 1024, 0)])
def test_attention_overlapping_query_ranges_do_not_wrap_the_units(cuda, B, T, page, hint):
    """Every other range takes all tokens again, over a million keys each: more units in all than 32 bits
    count, though no request for itself has. Nothing is computed, and the error says so."""
    g = _gen(cuda, 6)
    kc, q = _bf16(g, 1, page, 1, 64), _bf16(g, T, 64, 64)
    width = 1024
    tables = torch.zeros(B, width, dtype=torch.int32, device=cuda)
    seq = torch.full((B,), width * page, dtype=torch.int32, device=cuda)
    cu = torch.tensor([0, T] * (B // 2) + [0], dtype=torch.int32, device=cuda)
    out, lse = torch.full_like(q, 7.0), torch.full((T, 64), 7.0, device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    ws = ops.attention_workspace(cuda)
    ops.paged_attention(q, kc, kc, tables, seq, cu, out, max_q_len=hint, workspace=ws, lse=lse, err_word=err)
    assert err.item() == 6 and (out == 7.0).all() and (lse == 7.0).all()
    assert (ws == 0).all()  # and the workspace is as a call needs it


def test_page_tables_pages_near_2_31_tokens(cuda):
    """Tokens + page size past 2^31 (tables alone: no cache has such pages)."""
    for page in (2 ** 31 - 1, 2 ** 30):
        _tables_case(cuda, [5, 0, page - 60, page, 0], [1, 3, 50, 0, 0], page, 1)
        _tables_case(cuda, [5, page - 60], [3000, 50], page, 1, pad=2000, in_place=True)
    _tables_case(cuda, [2 ** 30 - 1, 2 ** 30 - 20], [2, 9], 2 ** 30 - 1, 2)
    one = dict(dtype=torch.int32, device=cuda)
    tables, lens, free, count = (torch.tensor(v, **one) for v in ([[3]], [2 ** 31 - 2], [-8, -8], [0]))
    ops.release_pages(torch.zeros(1, **one), lens, 2 ** 31 - 1, tables, free, count)
    assert free.tolist() == [3, -8] and count.item() == 1 and lens.item() == 0 and tables.item() == -1


def test_strides_of_dimensions_of_one_do_not_count(cuda):
    """One token out of a wider row, or one head: nothing is read at that stride, whatever it says."""
    g = _gen(cuda, 31)
    D, Hq = 64, 4
    ws = ops.attention_workspace(cuda)
    i32 = dict(dtype=torch.int32, device=cuda)
    cs = torch.cat([torch.ones(8, D, device=cuda)[:, :32], torch.zeros(8, 32, device=cuda)], 1)
    for Hkv in (1, 2):
        kc, vc = _bf16(g, 3, 16, Hkv, D), _bf16(g, 3, 16, Hkv, D)
        if Hkv == 1:
            kc, vc = (c.as_strided(c.shape, (16 * D, D, 3, 1)) for c in (kc, vc))
        qkv = _bf16(g, 1, (Hq + 2 * Hkv) * D)
        qkv = qkv.as_strided(qkv.shape, ((Hq + 2 * Hkv) * D + 5, 1))
        q, out = (_bf16(g, 1, Hq, D).as_strided((1, Hq, D), (7, D, 1)) for _ in range(2))
        ops.rope_cache_write(qkv, torch.zeros(1, **i32), torch.tensor([40], device=cuda), cs, kc, vc, q)
        x = qkv.view(Hq + 2 * Hkv, D)
        assert torch.equal(q[0], x[:Hq]) and torch.equal(kc[2, 8], x[Hq:Hq + Hkv])
        assert torch.equal(vc[2, 8], x[Hq + Hkv:])
        tables = torch.tensor([[1, 0, 2]], **i32)
        ops.paged_attention(q, kc, vc, tables, torch.tensor([41], **i32), torch.tensor([0, 1], **i32), out,
                            max_q_len=1, workspace=ws)
        want, _, tol, _ = _attention64(q, kc, vc, tables, [41], [0, 1], D ** -0.5, 0)
        _within(out, want, tol)


def test_attention_first_called_from_several_host_threads(cuda):
    """Through the C ABI (ctypes leaves the interpreter's lock), in a process that has not called it yet: each
    thread on a stream and a workspace of its own."""
    code = """
import ctypes, threading, torch
import tests.test_gpu_decoder_ops as t
from vllm_ascend_hust_latchmoe_b200 import _lib
dev, lib, P = torch.device('cuda', 0), _lib.load(), ctypes.c_void_p
g = t._gen(dev, 3)
kc, vc = t._bf16(g, 40, 16, 2, 64), t._bf16(g, 40, 16, 2, 64)
ids = torch.arange(40, dtype=torch.int32, device=dev).view(1, 40)
sizes = [(1, 300), (70, 600), (3, 640), (200, 200)] * 2
cases = []
for n, L in sizes:
    q = t._bf16(g, n, 8, 64)
    cases.append((q, torch.empty_like(q), torch.tensor([L], dtype=torch.int32, device=dev),
                  torch.tensor([0, n], dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev),
                  torch.zeros(200 << 20, dtype=torch.uint8, device=dev), torch.cuda.Stream()))
torch.cuda.synchronize()
gate, rcs = threading.Barrier(len(cases)), []
def work(q, out, seq, cu, err, ws, stream):
    p = [P(x.data_ptr()) for x in (q, kc, vc, ids, seq, cu, out, ws, err)]
    gate.wait()
    rc = lib.lm_paged_attention(p[0], 512, 64, p[1], 2048, 128, 64, p[2], 2048, 128, 64, 40, 16, p[3], 40, 40,
                                p[4], p[5], 1, q.shape[0], 8, 2, 64, q.shape[0], 0.125, 0, p[6], 512, 64, None, p[7],
                                ws.numel(), p[8], P(stream.cuda_stream))
    rcs.append((rc, rc and lib.lm_last_error()))
threads = [threading.Thread(target=work, args=c) for c in cases]
[x.start() for x in threads]
[x.join() for x in threads]
torch.cuda.synchronize()
assert rcs == [(0, 0)] * len(cases), rcs
for (q, out, *_), (n, L) in zip(cases, sizes):
    want, _, tol, _ = t._attention64(q, kc, vc, ids, [L], [0, n], 0.125, 0)
    t._within(out, want, tol)
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
