"""The paged decoder (chunked prefill, mixed steps, graph decode) against a plain fp32 forward pass of
the same weights over whole sequences.

All experts of the small model are active (top_k = experts), so that a near-tied router choice
cannot part two computations. Bar: every step of a layer rounds to bf16 (at most 2^-8 relative,
uniform rms 2^-8 / sqrt(12) of the binade, ten places a layer), so independent errors of two layers
sum to about sqrt(20) * 0.2 % = 1 %; logits are held to 3 % of their norm (8-bit activations and
weights of the QKV projection: 2^-4 in the place of 2^-8 there, 10 %)."""

import pytest
import torch

from vllm_ascend_hust_latchmoe_b200.decode_harness import DecoderShape
from vllm_ascend_hust_latchmoe_b200.paged_decoder import PagedKVCache, PagedMoEDecoder
from vllm_ascend_hust_latchmoe_b200.weight_layout import from_tiled

pytestmark = pytest.mark.gpu

TINY = DecoderShape(layers=2, hidden=256, heads=6, kv_heads=2, head_dim=64, experts=4, top_k=4,
                    intermediate=128, vocab=512)


def _make(cuda, **kw):
    args = dict(max_requests=3, max_len=160, max_tokens=200, page_size=16, seed=3, std=0.05)
    return PagedMoEDecoder(TINY, device=cuda, **{**args, **kw})


def _reference(dec, tokens):
    """Logits at every position of one sequence, fp32 and without a cache."""
    s, n = dec.s, len(tokens)

    def norm(x, w):
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()

    x = dec.embed[torch.tensor(tokens, device=dec.device)].float()
    cos, sin = dec.cos_sin[:n, None, :s.head_dim // 2], dec.cos_sin[:n, None, s.head_dim // 2:]

    def turn(t):
        a, b = t.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    mask = torch.ones(n, n, dtype=torch.bool, device=dec.device).tril()
    for i in range(s.layers):
        qkv = norm(x, dec.ln1[i]) @ dec.wqkv[i].float().t()
        q = turn(norm(qkv[:, :dec.qd].view(n, s.heads, -1), dec.q_norm[i]))
        k = turn(norm(qkv[:, dec.qd:dec.qd + dec.kvd].view(n, s.kv_heads, -1), dec.k_norm[i]))
        v = qkv[:, dec.qd + dec.kvd:].view(n, s.kv_heads, -1)
        k, v = (t.repeat_interleave(s.heads // s.kv_heads, 1) for t in (k, v))
        w = (torch.einsum("qhd,khd->hqk", q, k) * s.head_dim ** -0.5).masked_fill(~mask, -torch.inf).softmax(-1)
        x = x + torch.einsum("hqk,khd->qhd", w, v).reshape(n, -1) @ dec.wo[i].float().t()
        h = norm(x, dec.ln2[i])
        route = (h @ dec.gate[i].t()).softmax(-1)
        store = dec.runtime.host_layer(i)
        w13, w2 = from_tiled(store.w13).float(), from_tiled(store.w2).float()
        for e in range(s.experts):
            gate, up = (h @ w13[e].t()).chunk(2, -1)
            x = x + route[:, e:e + 1] * ((torch.nn.functional.silu(gate) * up) @ w2[e].t())
    return norm(x, dec.final_norm) @ dec.lm_head.float().t()


def _near(got, want, bar):
    err = (got.float() - want).norm() / want.norm()
    assert err <= bar, err.item()


@pytest.mark.parametrize("fp8", [False, True])
def test_chunks_and_mixed_steps_match_whole_sequences(cuda, fp8):
    dec = _make(cuda, fp8_qkv=fp8)
    bar = 0.10 if fp8 else 0.03
    g = torch.Generator().manual_seed(1)
    seqs = [torch.randint(TINY.vocab, (n,), generator=g).tolist() for n in (97, 33, 64)]
    want = [_reference(dec, s) for s in seqs]
    at = [0, 0, 0]
    for sizes in ((50, 1, 0), (1, 16, 64), (46, 15, 0), (0, 1, 0)):
        dec.step([s[a:a + n] for s, a, n in zip(seqs, at, sizes)])
        at = [a + n for a, n in zip(at, sizes)]
        for b, n in enumerate(sizes):
            if n:
                _near(dec.logits[b], want[b][at[b] - 1], bar)
    dec.cache.check_errors()
    assert at == [97, 33, 64] and dec.cache.lens.tolist() == at
    for layer in dec.moe:
        layer.check_device_errors()
    # the rows' pages come back, and the freed rows serve other requests
    held = dec.cache.free_count.item()
    dec.cache.release([0, 2])
    assert dec.cache.free_count.item() == held + 7 + 4
    dec.step([seqs[2], (), seqs[1]])
    _near(dec.logits[0], want[2][-1], bar)
    _near(dec.logits[2], want[1][-1], bar)
    dec.cache.check_errors()


def test_decode_graph_follows_its_own_tokens(cuda):
    dec = _make(cuda)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(TINY.vocab, (n,), generator=g).tolist() for n in (40, 7, 90)]
    out = dec.generate(prompts, 20, chunk=64)
    assert [len(o) for o in out] == [20, 20, 20] and dec._graph is not None
    for p, o in zip(prompts, out):  # teacher forcing: every token is the reference's best, or as good
        logits = _reference(dec, p + o[:-1])[len(p) - 1:]
        best = logits.max(-1).values
        chosen = logits[torch.arange(20, device=cuda), torch.tensor(o, device=cuda)]
        assert ((best - chosen) <= 0.06 * logits.norm(dim=-1) / TINY.vocab ** 0.5 * 4).all()
    dec.cache.release([0, 1, 2])
    assert dec.generate(prompts, 20, chunk=64) == out  # the graph again, on other pages
    dec.cache.release([0, 1, 2])
    assert dec.cache.free_count.item() == dec.cache.k[0].shape[0]


def test_running_out_of_pages_is_reported(cuda):
    dec = _make(cuda, num_pages=4)
    dec.step([list(range(40)), list(range(20)), [1]])
    with pytest.raises(RuntimeError, match="page"):
        dec.cache.check_errors()


def test_refusals(cuda):
    c = PagedKVCache(layers=1, num_pages=4, page_size=16, kv_heads=1, head_dim=64, max_requests=2,
                     max_len=64, max_tokens=8, device=cuda)
    for bad in ([1], [1, -1], [5, 4]):
        with pytest.raises(ValueError):
            c.set_new_lens(bad)
    dec = _make(cuda)
    with pytest.raises(ValueError):
        dec.generate([[1], [2]], 4, 8)
    with pytest.raises(ValueError):
        dec.generate([[1], [2], []], 4, 8)
    with pytest.raises(ValueError):
        dec.generate([[1], [2], [3]], 4, 199)


def test_tokens_outside_the_vocabulary_are_refused(cuda):
    """Before anything is launched: the embedding's rows are read at the tokens' numbers."""
    dec = _make(cuda)
    for bad in ([TINY.vocab], [3, -1], [-(2 ** 31)], [2 ** 40]):
        with pytest.raises(ValueError, match="token"):
            dec.step([[1, 2], bad, ()])
        with pytest.raises(ValueError, match="token"):
            dec.generate([[1, 2], bad, [5]], 4, 64)
    assert dec.cache.lens.tolist() == [0, 0, 0]
    dec.step([[0, TINY.vocab - 1], None, ()])
    dec.cache.check_errors()
    assert dec.cache.lens.tolist() == [2, 1, 0]
