"""What the decoder operators around the slot-bank MoE layer are measured on.

Four operators carry a decoder layer's attention half in serving:

* ``tables``     block tables, positions and slot maps of one step, from request lengths;
* ``rope_write`` per-head RMS norm and rotary embedding of a fused QKV projection's output, with
                 the new K and V written into the paged cache;
* ``attention``  attention of the step's new tokens (single tokens, chunks, whole prompts) over
                 the paged cache;
* ``norm``       residual addition and RMS norm, with bf16 or e4m3 + scales output.

``run`` computes them in elementary torch operations in 32 bits where ``own`` is false, and through
``vllm_ascend_hust_latchmoe_b200.decoder_ops`` where it is true.
"""

import math
import random

import torch

own = False

E4M3_MAX = 448.0
SCALE_FLOOR = 1e-12  # least |y| maximum that an e4m3 scale is made for
EPS = 1e-6


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a decode step of 64 requests: the smallest table build, repeated for every token
        dict(name="tables_decode_64", op="tables", requests=64, new=1, context=1280, page_size=16,
             singles=64, ragged=True),
        # a chunked-prefill step: 1021 requests, most of them decoding, the rest bringing prompts
        dict(name="tables_mixed_1021", op="tables", requests=1021, new=2048, context=8192,
             page_size=16, singles=1000, ragged=True),
        # one decode step of 16 requests of a 32-query-head, 4-kv-head layer with q/k norms
        dict(name="rope_decode_16", op="rope_write", tokens=16, q_heads=32, kv_heads=4, head_dim=128,
             rot_dim=128, page_size=16, qk_norm=True, interleaved=False),
        # a 4096-token prefill of the same layer
        dict(name="rope_prefill_4096", op="rope_write", tokens=4096, q_heads=32, kv_heads=4,
             head_dim=128, rot_dim=128, page_size=16, qk_norm=True, interleaved=False),
        # the norm in front of a decode layer's projections, 16 tokens
        dict(name="norm_decode_16", op="norm", tokens=16, hidden=2048, residual=True, fp8=False,
             group=0),
        # a ragged prefill chunk's norm
        dict(name="norm_prefill_4093", op="norm", tokens=4093, hidden=2048, residual=True, fp8=False,
             group=0),
        # a large prefill's norm in front of an e4m3 projection with scales per 128 columns
        dict(name="norm_fp8_16384", op="norm", tokens=16384, hidden=4096, residual=True, fp8=True,
             group=128),
        # one token of one request after a 1024-token prompt and some new tokens
        dict(name="attn_decode_1", op="attention", requests=1, new=1, context=1151, singles=1,
             ragged=False, q_heads=32, kv_heads=4, head_dim=128, page_size=16, window=0),
        # a decode step of 64 requests with contexts of up to 8192 tokens, 16 query heads a kv head
        dict(name="attn_decode_64", op="attention", requests=64, new=1, context=8191, singles=64,
             ragged=True, q_heads=64, kv_heads=4, head_dim=128, page_size=16, window=0),
        # two requests with very long contexts: work split over the sequence
        dict(name="attn_decode_long", op="attention", requests=2, new=1, context=131071, singles=2,
             ragged=False, q_heads=32, kv_heads=4, head_dim=128, page_size=64, window=0),
        # a mixed step: decoding requests and ragged prompts, 7 query heads a kv head of 64
        dict(name="attn_mixed_8", op="attention", requests=8, new=1000, context=3000, singles=4,
             ragged=True, q_heads=14, kv_heads=2, head_dim=64, page_size=32, window=0),
        # a 4096-token chunk after 12288 cached tokens
        dict(name="attn_chunk_4096", op="attention", requests=1, new=4096, context=12288, singles=0,
             ragged=False, q_heads=32, kv_heads=4, head_dim=128, page_size=16, window=0),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.499)))))))


def draw(rng):
    op = rng.choice(["tables", "rope_write", "norm", "attention", "attention"])
    page = rng.choice([16, 32, 64, 128])
    if op == "tables":
        B = _log(rng, 1, 1024)
        new = _log(rng, 1, 4096)
        singles = B if new == 1 else rng.randint(max(0, B - 16384 // new), B)
        return dict(op=op, requests=B, new=new, context=_log(rng, 1, 16384), page_size=page,
                    singles=singles, ragged=True)
    if op == "rope_write":
        D = rng.choice([64, 128])
        kv = rng.choice([1, 2, 4, 8])
        return dict(op=op, tokens=_log(rng, 1, 4096), q_heads=kv * rng.choice([1, 2, 4, 5, 7, 8]),
                    kv_heads=kv, head_dim=D, rot_dim=rng.choice([D, D // 2]), page_size=page,
                    qk_norm=rng.random() < 0.5, interleaved=rng.random() < 0.3)
    if op == "norm":
        fp8 = rng.random() < 0.5
        H = rng.choice([64, 1000, 1001, 1408, 2048, 2880, 4096, 5120, 7168, 8192])
        group = 128 if fp8 and H % 128 == 0 and rng.random() < 0.5 else 0
        return dict(op=op, tokens=_log(rng, 1, 16384 * 4096 // max(H, 4096)), hidden=H,
                    residual=rng.random() < 0.8, fp8=fp8, group=group)
    D = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8])
    q = kv * rng.choice([1, 2, 4, 5, 7, 8, 16])
    kind = rng.choice(["decode", "chunk", "mixed"])
    B = _log(rng, 1, 64) if kind == "decode" else _log(rng, 1, 8)
    new = 1 if kind == "decode" else _log(rng, 2, 4096)
    context = _log(rng, 1, 131072)
    # at most the listed cases' work: cache bytes, and scores (which the plain form holds)
    while B * context * kv * D * 4 > 500e6 or B * q * new * (context + new) > 32 * 4096 * 14000:
        if B > 2:
            B -= 1
        elif new > 64:
            new = new * 3 // 4
        else:
            context = context * 3 // 4
    singles = B if kind == "decode" else 0 if kind == "chunk" else rng.randint(0, B)
    return dict(op=op, requests=B, new=new, context=context, singles=singles, ragged=True, q_heads=q,
                kv_heads=kv, head_dim=D, page_size=page,
                window=_log(rng, 1, context + new) if rng.random() < 0.25 else 0)


def _lens(case):
    """(cached, new) lengths of the case's requests: a property of the case, not of the seed."""
    key = {k: v for k, v in case.items() if k != "name"}
    rng = random.Random(repr(sorted(key.items())))
    B, ragged = case["requests"], case["ragged"]
    cached = [case["context"] if not ragged or i == 0 else rng.randint(0, case["context"]) for i in range(B)]
    new = [1 if i < case["singles"] else
           case["new"] if not ragged or i == B - 1 else rng.randint(max(1, case["new"] // 4), case["new"])
           for i in range(B)]
    return cached, new


def _pages(n, page):
    return -(-n // page)


# ------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dev = torch.device("cuda")

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * std).to(torch.bfloat16)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=dev)

    def kept(*shape, dtype):  # a buffer that a serving loop owns and reuses
        return torch.zeros(*shape, dtype=dtype, device=dev)

    op, s = case["op"], {"case": case}
    if op == "norm":
        T, H = case["tokens"], case["hidden"]
        s.update(x=normal(T, H), weight=normal(H, std=0.1) + 1.0)
        if case["residual"]:
            # a residual stream: larger than a layer's output, with a few outlying columns
            spread = torch.ones(H, device=dev)
            spread[torch.randint(H, (max(1, H // 256),), device=dev, generator=g)] = 20.0
            s["residual"] = (torch.randn(T, H, device=dev, generator=g) * spread * 3.0).to(torch.bfloat16)
            s["residual_out"] = kept(T, H, dtype=torch.bfloat16)
        if case["fp8"]:
            s["out"] = kept(T, H, dtype=torch.float8_e4m3fn)
            s["scales"] = kept(T, H // case["group"] if case["group"] else 1, dtype=torch.float32)
        else:
            s["out"] = kept(T, H, dtype=torch.bfloat16)
        return s
    if op == "tables":
        cached, new = _lens(case)
        page, B, T = case["page_size"], case["requests"], sum(new)
        have = [_pages(c, page) for c in cached]
        total = [_pages(c + n, page) for c, n in zip(cached, new)]
        width = _pages(case["context"] + case["new"], page)
        pool = torch.randperm(sum(total) + 17, device=dev, generator=g, dtype=torch.int32)
        tables = torch.full((B, width), -1, dtype=torch.int32, device=dev)
        held = torch.arange(width, device=dev)[None, :] < ints(have)[:, None]
        tables[held] = pool[:sum(have)]
        s.update(cached=ints(cached), new=ints(new), tables=tables, page=page, tokens=T,
                 free=pool[sum(have):].clone(), free_count=ints([len(pool) - sum(have)]),
                 free_left=kept(1, dtype=torch.int32), seq_lens=kept(B, dtype=torch.int32),
                 cu_q=kept(B + 1, dtype=torch.int32), positions=kept(T, dtype=torch.int32),
                 slots=kept(T, dtype=torch.int64))
        return s
    Hq, Hkv, D, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page_size"]
    if op == "rope_write":
        T, R = case["tokens"], case["rot_dim"]
        pages = _pages(T, page) + 3
        start = int(torch.randint(4096, (1,), device=dev, generator=g))
        angle = (torch.arange(8192, device=dev, dtype=torch.float64)[:, None]
                 * 1e6 ** (-torch.arange(0, R, 2, device=dev, dtype=torch.float64) / R)[None, :])
        order = torch.randperm(pages, device=dev, generator=g)
        t = torch.arange(T, device=dev)
        s.update(qkv=normal(T, (Hq + 2 * Hkv) * D), page=page,
                 positions=((start + t) % 8192).to(torch.int32), slots=order[t // page] * page + t % page,
                 cos_sin=torch.cat([angle.cos(), angle.sin()], 1).float(),
                 k_cache=normal(pages, page, Hkv, D), v_cache=normal(pages, page, Hkv, D),
                 q=kept(T, Hq, D, dtype=torch.bfloat16), q_weight=None, k_weight=None)
        if case["qk_norm"]:
            s.update(q_weight=normal(D, std=0.1) + 1.0, k_weight=normal(D, std=0.1) + 1.0)
        return s
    cached, new = _lens(case)
    B, T = case["requests"], sum(new)
    total = [_pages(c + n, page) for c, n in zip(cached, new)]
    pool = torch.randperm(sum(total) + 5, device=dev, generator=g, dtype=torch.int32)
    tables = torch.full((B, max(total)), -1, dtype=torch.int32, device=dev)
    tables[torch.arange(max(total), device=dev)[None, :] < ints(total)[:, None]] = pool[:sum(total)]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    # heads differ in how sharply they attend
    sharp = torch.exp2(2.0 * torch.rand(Hq, 1, device=dev, generator=g))
    s.update(q=(torch.randn(T, Hq, D, device=dev, generator=g) * sharp).to(torch.bfloat16),
             k_cache=normal(len(pool), page, Hkv, D), v_cache=normal(len(pool), page, Hkv, D),
             tables=tables, seq_lens=ints([c + n for c, n in zip(cached, new)]), cu_q=ints(starts),
             max_q=max(new), window=case["window"], scale=1.0 / math.sqrt(D),
             out=kept(T, Hq, D, dtype=torch.bfloat16), lse=kept(T, Hq, dtype=torch.float32))
    return s


# ------------------------------------------------------------------------------------ one pass
_workspace = None  # one attention workspace per process, as a serving loop keeps it


def run(s):
    op = s["case"]["op"]
    if own:
        return _OWN[op](s)
    return _PLAIN[op](s)


def _own_norm(s):
    from vllm_ascend_hust_latchmoe_b200 import decoder_ops as ops

    if s["case"]["fp8"]:
        ops.add_rms_norm(s["x"], s["weight"], EPS, residual=s.get("residual"),
                         residual_out=s.get("residual_out"), out_fp8=s["out"], scales=s["scales"],
                         group_size=s["case"]["group"])
        return {"y": s["out"], "scales": s["scales"], "residual": s.get("residual_out")}
    ops.add_rms_norm(s["x"], s["weight"], EPS, residual=s.get("residual"),
                     residual_out=s.get("residual_out"), out=s["out"])
    return {"y": s["out"], "residual": s.get("residual_out")}


def _own_tables(s):
    from vllm_ascend_hust_latchmoe_b200 import decoder_ops as ops

    ops.build_page_tables(s["cached"], s["new"], s["page"], s["tables"], s["free"], s["free_count"],
                          seq_lens=s["seq_lens"], cu_q=s["cu_q"], positions=s["positions"],
                          slot_mapping=s["slots"], free_count_out=s["free_left"])
    return {"tables": s["tables"], "seq_lens": s["seq_lens"], "cu_q": s["cu_q"],
            "positions": s["positions"], "slots": s["slots"], "free_left": s["free_left"]}


def _own_rope(s):
    from vllm_ascend_hust_latchmoe_b200 import decoder_ops as ops

    ops.rope_cache_write(s["qkv"], s["positions"], s["slots"], s["cos_sin"], s["k_cache"], s["v_cache"],
                         s["q"], q_norm_weight=s["q_weight"], k_norm_weight=s["k_weight"], eps=EPS,
                         interleaved=s["case"]["interleaved"])
    return {"q": s["q"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_attention(s):
    from vllm_ascend_hust_latchmoe_b200 import decoder_ops as ops

    global _workspace
    if _workspace is None:
        _workspace = ops.attention_workspace(s["q"].device)
    ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["seq_lens"], s["cu_q"],
                        s["out"], max_q_len=s["max_q"], scale=s["scale"], window=s["window"],
                        lse=s["lse"], workspace=_workspace)
    return {"out": s["out"], "lse": s["lse"]}


def _plain_norm(s):
    x = s["x"].float()
    if "residual" in s:
        x = x + s["residual"].float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["weight"].float()
    kept = x.to(torch.bfloat16) if "residual" in s else None
    if not s["case"]["fp8"]:
        return {"y": y.to(torch.bfloat16), "residual": kept}
    T, H = y.shape
    groups = y.view(T, -1, s["case"]["group"] or H)
    scales = groups.abs().amax(-1).clamp(min=SCALE_FLOOR) / E4M3_MAX
    return {"y": (groups / scales[..., None]).view(T, H).to(torch.float8_e4m3fn), "scales": scales,
            "residual": kept}


def _plain_tables(s):
    cached, new, page, tables = s["cached"], s["new"], s["page"], s["tables"]
    have, total = (cached + page - 1) // page, (cached + new + page - 1) // page
    taken = (total - have).cumsum(0)
    cols = torch.arange(tables.shape[1], device=tables.device)[None, :]
    at = s["free_count"] - 1 - ((taken - total + have)[:, None] + cols - have[:, None])
    fresh = (cols >= have[:, None]) & (cols < total[:, None])
    tables = torch.where(fresh, s["free"][at.clamp(0, s["free"].numel() - 1)], tables)
    cu_q = torch.cat([torch.zeros_like(s["free_count"]), new.cumsum(0).to(torch.int32)])
    t = torch.arange(s["tokens"], dtype=torch.int32, device=tables.device)
    b = torch.searchsorted(cu_q[1:].contiguous(), t, right=True)
    positions = cached[b] + t - cu_q[b]
    slots = tables[b, positions // page].long() * page + positions % page
    return {"tables": tables, "seq_lens": cached + new, "cu_q": cu_q, "positions": positions,
            "slots": slots, "free_left": (s["free_count"] - taken[-1:]).to(torch.int32)}


def _plain_heads(x, weight, cos, sin, interleaved):
    """Norm (where there is a weight) and rotary embedding of x [T, heads, D] in 32 bits."""
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    R = 2 * cos.shape[-1]
    turned, rest = x[..., :R], x[..., R:]
    cos, sin = cos[:, None, :], sin[:, None, :]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :R // 2], turned[..., R // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1).to(torch.bfloat16)


def _plain_rope(s):
    c = s["case"]
    T, Hq, Hkv, D = c["tokens"], c["q_heads"], c["kv_heads"], c["head_dim"]
    x = s["qkv"].float().view(T, Hq + 2 * Hkv, D)
    cs = s["cos_sin"][s["positions"].long()]
    cos, sin = cs[:, :c["rot_dim"] // 2], cs[:, c["rot_dim"] // 2:]
    q = _plain_heads(x[:, :Hq], s["q_weight"], cos, sin, c["interleaved"])
    k = _plain_heads(x[:, Hq:Hq + Hkv], s["k_weight"], cos, sin, c["interleaved"])
    at = (s["slots"] // s["page"], s["slots"] % s["page"])
    s["k_cache"][at] = k
    s["v_cache"][at] = x[:, Hq + Hkv:].to(torch.bfloat16)
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s):
    q, tables, seq, cu = s["q"], s["tables"], s["seq_lens"].long(), s["cu_q"].long()
    T, Hq, D = q.shape
    B, Hkv = tables.shape[0], s["k_cache"].shape[2]
    new = cu[1:] - cu[:-1]
    i = torch.arange(s["max_q"], device=q.device)
    rows = (cu[:-1, None] + i).clamp(max=T - 1)
    qp = q[rows].float().view(B, s["max_q"], Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4)
    at = tables.clamp(min=0).long()
    k = s["k_cache"][at].flatten(1, 2).float().permute(0, 2, 3, 1)
    v = s["v_cache"][at].flatten(1, 2).float().permute(0, 2, 1, 3)
    L = k.shape[-1]
    w = torch.matmul(qp.reshape(B, Hkv, -1, D), k).mul_(s["scale"]).view(B, Hkv, -1, s["max_q"], L)
    here = (seq - new)[:, None] + i
    j = torch.arange(L, device=q.device)
    seen = (j <= here[..., None]) & (j < seq[:, None, None]) & (i < new[:, None])[..., None]
    if s["window"]:
        seen &= j > here[..., None] - s["window"]
    w.masked_fill_(~seen[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    w.sub_(top).exp_()
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w.view(B, Hkv, -1, L), v).view(B, Hkv, -1, s["max_q"], D)
    out = out / torch.where(total == 0, torch.ones_like(total), total)
    lse = (top + total.log())[..., 0]
    t = torch.arange(T, device=q.device)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    r = t - cu[b]
    return {"out": out.permute(0, 3, 1, 2, 4)[b, r].reshape(T, Hq, D).to(torch.bfloat16),
            "lse": lse.permute(0, 3, 1, 2)[b, r].reshape(T, Hq)}


_OWN = {"norm": _own_norm, "tables": _own_tables, "rope_write": _own_rope, "attention": _own_attention}
_PLAIN = {"norm": _plain_norm, "tables": _plain_tables, "rope_write": _plain_rope,
          "attention": _plain_attention}


# ------------------------------------------------------------------------------------ floors
def work(case):
    op = case["op"]
    if op == "norm":
        n = case["tokens"] * case["hidden"]
        groups = case["hidden"] // case["group"] if case["group"] else 1
        return {"bytes": n * (2 + (4 if case["residual"] else 0) + (1 if case["fp8"] else 2))
                + case["hidden"] * 2 + (case["tokens"] * groups * 4 if case["fp8"] else 0),
                "flops": 5 * n}
    if op == "rope_write":
        T, heads = case["tokens"], case["q_heads"] + 2 * case["kv_heads"]
        n = T * heads * case["head_dim"]
        return {"bytes": 4 * n + T * (12 + 4 * case["rot_dim"]), "flops": 8 * n}
    cached, new = _lens(case)
    page, B, T = case["page_size"], case["requests"], sum(new)
    if op == "tables":
        fresh = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(cached, new))
        return {"bytes": 16 * B + 8 * fresh + 12 * T + 8, "flops": 4 * T}
    Hq, Hkv, D, window = case["q_heads"], case["kv_heads"], case["head_dim"], case["window"]
    pairs = keys = 0
    for c, n in zip(cached, new):
        if window:
            full = max(0, min(n, c + n - window + 1))  # rows whose window is full; the first ones are not
            first = n - full
            pairs += full * window + first * c + first * (first + 1) // 2
            keys += min(c + n, window + n - 1)
        else:
            pairs += n * c + n * (n + 1) // 2
            keys += c + n
    return {"bytes": keys * Hkv * D * 4 + T * Hq * (4 * D + 4) + 4 * _pages(keys, page) + 8 * B,
            "flops": 4 * D * Hq * pairs}


# ------------------------------------------------------------------------------------ 64 bits
def _round_e4m3(v):
    """The nearest e4m3 value (ties to even) of values of at most 448 in magnitude."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=-6) - 3)
    return torch.round(v / step) * step


def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "norm":
        z = s["x"].double()
        if case["residual"]:
            z = z + s["residual"].double()
        y = z / (z.pow(2).sum(1, keepdim=True) / case["hidden"] + EPS).sqrt() * s["weight"].double()
        kept = z if case["residual"] else None
        if not case["fp8"]:
            return {"y": y, "residual": kept}
        parts = y.split(case["group"] or case["hidden"], dim=1)
        scales = torch.stack([p.abs().max(1).values.clamp(min=SCALE_FLOOR) / E4M3_MAX for p in parts], 1)
        y8 = torch.cat([_round_e4m3(p / scales[:, n, None]) for n, p in enumerate(parts)], 1)
        return {"y": y8, "scales": scales, "residual": kept}
    Hq, Hkv, D = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rope_write":
        T, R = case["tokens"], case["rot_dim"]
        heads = s["qkv"].double().view(T, Hq + 2 * Hkv, D)
        c = s["cos_sin"][s["positions"].long()].double()
        first = torch.arange(0, R, 2) if case["interleaved"] else torch.arange(R // 2)
        second = first + (1 if case["interleaved"] else R // 2)
        new = []
        for h in range(Hq + Hkv):
            z, wt = heads[:, h], s["q_weight"] if h < Hq else s["k_weight"]
            if wt is not None:
                z = z / (z.pow(2).sum(1, keepdim=True) / D + EPS).sqrt() * wt.double()
            turn = torch.complex(z[:, first], z[:, second]) * torch.complex(c[:, :R // 2], c[:, R // 2:])
            z = z.clone()
            z[:, first], z[:, second] = turn.real, turn.imag
            new.append(z)
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        flat = s["slots"]
        kc.view(-1, Hkv, D)[flat] = torch.stack(new[Hq:], 1)
        vc.view(-1, Hkv, D)[flat] = heads[:, Hq + Hkv:]
        return {"q": torch.stack(new[:Hq], 1), "k_cache": kc, "v_cache": vc}
    cached, new = _lens(case)
    out = torch.zeros(sum(new), Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((sum(new), Hq), -math.inf, dtype=torch.float64, device="cuda")
    at, page, G = 0, case["page_size"], Hq // Hkv
    for b in range(case["requests"]):
        L = cached[b] + new[b]
        held = s["tables"][b, :_pages(L, page)].long()
        keys = s["k_cache"][held].reshape(-1, Hkv, D)[:L].double()
        values = s["v_cache"][held].reshape(-1, Hkv, D)[:L].double()
        for lo in range(0, new[b], 512):
            hi = min(new[b], lo + 512)
            p = torch.arange(cached[b] + lo, cached[b] + hi, device="cuda")[:, None]
            j = torch.arange(L, device="cuda")[None, :]
            hidden = (j > p) | (j <= p - case["window"]) if case["window"] else j > p
            for h in range(Hq):
                z = s["q"][at + lo:at + hi, h].double() @ keys[:, h // G].t() * s["scale"]
                z[hidden] = -math.inf
                lse[at + lo:at + hi, h] = torch.logsumexp(z, 1)
                out[at + lo:at + hi, h] = torch.softmax(z, 1) @ values[:, h // G]
        at += new[b]
    return {"out": out, "lse": lse}
