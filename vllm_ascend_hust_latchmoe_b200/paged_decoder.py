"""A MoE decoder served over a paged KV cache: chunked prefill and batched decode in one loop.

    python -m vllm_ascend_hust_latchmoe_b200.paged_decoder --layers 8 --requests 16 --new-tokens 64

:class:`PagedKVCache` holds every layer's K and V pages and the step's tables, all on the device;
:class:`PagedMoEDecoder` runs a Qwen3-30B-A3B-shaped stack (random weights) with the operators of
:mod:`.decoder_ops` around the slot-bank MoE layer:

    page tables -> per layer: residual + RMS norm (e4m3 with ``fp8_qkv``) -> QKV projection ->
    q/k norm + rotary embedding + cache write -> paged attention -> output projection ->
    residual + RMS norm -> router -> grouped expert MLP (experts resident in HBM)

Each step takes any mix of prompt chunks and single tokens (:meth:`PagedMoEDecoder.step`); a step
in which every request decodes is replayed from one CUDA graph, since lengths, tables and free
pages live on the device. The projections are plain library GEMMs.
"""

from __future__ import annotations

import argparse
import json
import time
from collections.abc import Sequence

import torch

from . import _lib, decoder_ops as ops
from .config import MoeOffloadConfig
from .decode_harness import DecoderShape
from .layer import SlotBankMoE
from .moe_offload.runtime import MoeOffloadRuntime


class PagedKVCache:
    """K and V pages of ``layers`` layers with one set of block tables, lengths and free pages.

    A request is a row. ``set_new_lens`` says how many tokens each row gets in the next step,
    ``build`` grants their pages and fills the step's tables (capturable), ``release`` gives the
    rows' pages back. ``lens`` are the rows' lengths, the new tokens included after ``build``."""

    def __init__(self, *, layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int,
                 max_requests: int, max_len: int, max_tokens: int,
                 device: torch.device | str = "cuda") -> None:
        d, i32 = torch.device(device), torch.int32
        shape = (num_pages, page_size, kv_heads, head_dim)
        self.page_size, self.max_requests, self.max_tokens = page_size, max_requests, max_tokens
        self.k = [torch.zeros(shape, dtype=torch.bfloat16, device=d) for _ in range(layers)]
        self.v = [torch.zeros(shape, dtype=torch.bfloat16, device=d) for _ in range(layers)]
        width = -(-max_len // page_size)
        self.block_tables = torch.full((max_requests, width), -1, dtype=i32, device=d)
        self.free_pages = torch.arange(num_pages, dtype=i32, device=d)
        self.free_count = torch.full((1,), num_pages, dtype=i32, device=d)
        self.lens = torch.zeros(max_requests, dtype=i32, device=d)
        self.new_lens = torch.zeros(max_requests, dtype=i32, device=d)
        self.cu_q = torch.zeros(max_requests + 1, dtype=i32, device=d)
        self.positions = torch.zeros(max_tokens, dtype=i32, device=d)
        self.slot_mapping = torch.zeros(max_tokens, dtype=torch.int64, device=d)
        self.err = torch.zeros(1, dtype=i32, device=d)

    def set_new_lens(self, new_lens: Sequence[int]) -> int:
        """The next step's token counts, one per row; returns their sum."""
        total = sum(new_lens)
        if len(new_lens) != self.max_requests or min(new_lens, default=0) < 0:
            raise ValueError(f"one count of at least 0 for each of the {self.max_requests} rows")
        if total > self.max_tokens:
            raise ValueError(f"{total} new tokens: a step takes at most {self.max_tokens}")
        self.new_lens.copy_(torch.tensor(new_lens, dtype=torch.int32))
        return total

    def build(self, tokens: int) -> None:
        """Pages, lengths, query offsets, positions and slots of a step of ``tokens`` tokens."""
        ops.build_page_tables(self.lens, self.new_lens, self.page_size, self.block_tables,
                              self.free_pages, self.free_count, seq_lens=self.lens, cu_q=self.cu_q,
                              positions=self.positions[:tokens],
                              slot_mapping=self.slot_mapping[:tokens], err_word=self.err)

    def release(self, rows: Sequence[int]) -> None:
        rows_dev = torch.tensor(list(rows), dtype=torch.int32).to(self.lens.device)
        ops.release_pages(rows_dev, self.lens, self.page_size, self.block_tables, self.free_pages,
                          self.free_count, self.err)

    def check_errors(self, where: str = "PagedKVCache") -> None:
        """Raise if a step ran out of pages or met a bad length (waits for the device)."""
        _lib.raise_on_device_error(self.err, where)


class PagedMoEDecoder:
    def __init__(self, shape: DecoderShape, *, max_requests: int, max_len: int, max_tokens: int,
                 page_size: int = 16, num_pages: int | None = None, fp8_qkv: bool = False,
                 device: torch.device | str = "cuda", seed: int = 0, std: float = 0.02) -> None:
        self.s = s = shape
        d = torch.device(device)
        self.device, self.max_requests, self.max_tokens = d, max_requests, max_tokens
        g = torch.Generator(device=d)
        g.manual_seed(seed)

        def rand(*size, scale=std):
            return (torch.randn(*size, device=d, generator=g) * scale).to(torch.bfloat16)

        H, D, L, I = s.hidden, s.head_dim, s.layers, s.intermediate
        self.qd, self.kvd = s.heads * D, s.kv_heads * D
        self.embed = rand(s.vocab, H, scale=1.0)
        self.lm_head = rand(s.vocab, H)
        self.final_norm = rand(H, scale=0.1) + 1
        self.ln1, self.ln2 = ([rand(H, scale=0.1) + 1 for _ in range(L)] for _ in range(2))
        self.q_norm, self.k_norm = ([rand(D, scale=0.1) + 1 for _ in range(L)] for _ in range(2))
        self.wqkv = [rand(self.qd + 2 * self.kvd, H) for _ in range(L)]
        self.wo = [rand(H, self.qd) for _ in range(L)]
        self.gate = [rand(s.experts, H).float() for _ in range(L)]
        self.fp8_qkv = bool(fp8_qkv)
        if self.fp8_qkv:  # e4m3 weights with a scale per output column
            self.wqkv8 = []
            for w in self.wqkv:
                scale = w.float().abs().amax(1, keepdim=True) / 448
                self.wqkv8.append(((w.float() / scale).to(torch.float8_e4m3fn), scale.t().contiguous()))
        inv = s.rope_theta ** (-torch.arange(0, D, 2, device=d, dtype=torch.float64) / D)
        angle = torch.arange(max_len, device=d, dtype=torch.float64)[:, None] * inv[None, :]
        self.cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float()

        self.runtime = MoeOffloadRuntime(MoeOffloadConfig(enabled=True, num_slots=1))
        self.moe = []
        for i in range(L):  # experts resident in HBM, in the bank's tiled order
            self.runtime.register_layer_with_store(i, rand(s.experts, 2 * I, H), rand(s.experts, H, I),
                                                   slot_device=d, num_slots=1)
            self.moe.append(SlotBankMoE(self.runtime, i, hidden_size=H, intermediate_size=I,
                                        num_experts=s.experts, top_k=s.top_k, max_tokens=max_tokens,
                                        device=d))
        pages = num_pages or max_requests * -(-max_len // page_size)
        self.cache = PagedKVCache(layers=L, num_pages=pages, page_size=page_size,
                                  kv_heads=s.kv_heads, head_dim=D, max_requests=max_requests,
                                  max_len=max_len, max_tokens=max_tokens, device=d)
        self.workspace = ops.attention_workspace(d)

        def rows(n, dtype=torch.bfloat16):
            return torch.zeros(max_tokens, n, dtype=dtype, device=d)

        self.residual, self.normed, self.delta = rows(H), rows(H), rows(H)
        self.normed8, self.scales = rows(H, torch.float8_e4m3fn), rows(1, torch.float32)
        self.qkv = rows(self.qd + 2 * self.kvd)
        self.q, self.attn = rows(self.qd), rows(self.qd)
        self.next_token = torch.zeros(max_requests, dtype=torch.int64, device=d)
        self.logits = torch.zeros(max_requests, s.vocab, dtype=torch.bfloat16, device=d)
        self._graph: torch.cuda.CUDAGraph | None = None

    # -------------------------------------------------------------------------------- a step
    def _qkv(self, i: int, T: int, residual: torch.Tensor | None, x: torch.Tensor) -> torch.Tensor:
        """Residual addition, norm and the QKV projection of layer ``i``."""
        qkv = self.qkv[:T]
        if not self.fp8_qkv:
            h = self.normed[:T]
            ops.add_rms_norm(x, self.ln1[i], residual=residual, residual_out=self.residual[:T], out=h)
            return torch.mm(h, self.wqkv[i].t(), out=qkv)
        h, scale = self.normed8[:T], self.scales[:T]
        ops.add_rms_norm(x, self.ln1[i], residual=residual, residual_out=self.residual[:T], out_fp8=h,
                         scales=scale)
        w, w_scale = self.wqkv8[i]
        return torch._scaled_mm(h, w.t(), scale_a=scale, scale_b=w_scale, out_dtype=torch.bfloat16, out=qkv)

    def _forward(self, tokens: torch.Tensor, T: int, max_q: int) -> None:
        """Tables, all layers and the next token of every row, from fixed buffers on."""
        s, c = self.s, self.cache
        c.build(T)
        delta, residual = self.delta[:T], self.residual[:T]
        x = self.embed.index_select(0, tokens)
        q, attn = (t[:T].view(T, s.heads, s.head_dim) for t in (self.q, self.attn))
        for i in range(s.layers):
            qkv = self._qkv(i, T, None if i == 0 else residual, x)
            ops.rope_cache_write(qkv, c.positions[:T], c.slot_mapping[:T], self.cos_sin, c.k[i], c.v[i],
                                 q, q_norm_weight=self.q_norm[i], k_norm_weight=self.k_norm[i],
                                 err_word=c.err)
            ops.paged_attention(q, c.k[i], c.v[i], c.block_tables, c.lens, c.cu_q, attn,
                                max_q_len=max_q, workspace=self.workspace, err_word=c.err)
            torch.mm(self.attn[:T], self.wo[i].t(), out=delta)
            h = self.normed[:T]
            ops.add_rms_norm(delta, self.ln2[i], residual=residual, residual_out=residual, out=h)
            self.moe[i].route(h, torch.mm(h.float(), self.gate[i].t()))
            x = self.moe[i].mlp_resident(h, T)
        h = self.normed[:T]
        ops.add_rms_norm(x, self.final_norm, residual=residual, residual_out=residual, out=h)
        last = (c.cu_q[1:] - 1).clamp(min=0).long()  # a row without new tokens takes any other's
        torch.mm(h.index_select(0, last), self.lm_head.t(), out=self.logits)
        self.next_token.copy_(self.logits.argmax(-1))

    def _check_tokens(self, rows: Sequence[Sequence[int] | None]) -> None:
        """The embedding's rows are read at these numbers."""
        for r in rows:
            if r is not None and len(r) and not 0 <= min(r) <= max(r) < self.s.vocab:
                raise ValueError(f"a token outside 0 .. {self.s.vocab - 1}")

    def step(self, rows: Sequence[Sequence[int] | None]) -> None:
        """One step: ``rows[b]`` is row b's next prompt chunk, or None for the token that the last
        step gave it, or () for nothing. Afterwards ``logits`` and ``next_token`` hold every row's
        (rows without new tokens: undefined)."""
        self._check_tokens(rows)
        new = [1 if r is None else len(r) for r in rows]
        T = self.cache.set_new_lens(new)
        if T == 0:
            return
        if T == self.max_requests and all(r is None for r in rows):
            self._decode()
            return
        flat = [t for b, r in enumerate(rows) for t in ((-1 - b,) if r is None else r)]
        flat = torch.tensor(flat).to(self.device)
        tokens = torch.where(flat < 0, self.next_token[(-1 - flat).clamp(min=0)], flat)
        self._forward(tokens, T, max(new))

    def _decode(self) -> None:
        """One token for every row, replayed from a graph (the first time: captured)."""
        if self._graph is None:
            # the libraries' lazy set-up happens outside the capture, on rows that get no tokens
            kept = self.next_token.clone(), self.cache.new_lens.clone()
            self.cache.new_lens.zero_()
            self._forward(self.next_token, self.max_requests, 1)
            self.next_token.copy_(kept[0])
            self.cache.new_lens.copy_(kept[1])
            torch.cuda.synchronize()
            self._graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self._graph):
                self._forward(self.next_token, self.max_requests, 1)
        self._graph.replay()

    # ---------------------------------------------------------------------------- generation
    def generate(self, prompts: Sequence[Sequence[int]], new_tokens: int, chunk: int) -> list[list[int]]:
        """Greedy generation: prompts enter in chunks, at most ``chunk`` prompt tokens a step, beside
        the rows that decode already."""
        if len(prompts) != self.max_requests or any(len(p) == 0 for p in prompts):
            raise ValueError(f"{self.max_requests} prompts of at least a token are wanted")
        self._check_tokens(prompts)
        if chunk < 1 or chunk + self.max_requests > self.max_tokens:
            raise ValueError("chunk + requests must fit a step's tokens")
        taken, made = [0] * len(prompts), [0] * len(prompts)
        out: list[torch.Tensor] = []
        who: list[list[int]] = []
        while min(made) < new_tokens:
            room, rows = chunk, []
            for b, prompt in enumerate(prompts):
                if taken[b] == len(prompt):
                    rows.append(None if made[b] < new_tokens else ())
                    continue
                n = min(room, len(prompt) - taken[b])
                rows.append(prompt[taken[b]:taken[b] + n])
                taken[b] += n
                room -= n
            self.step(rows)
            gave = [b for b, r in enumerate(rows) if taken[b] == len(prompts[b]) and (r is None or len(r))]
            for b in gave:
                made[b] += 1
            out.append(self.next_token.clone())
            who.append(gave)
        tokens = torch.stack(out).cpu().tolist()
        self.cache.check_errors("generate")
        for layer in self.moe:
            layer.check_device_errors("generate")
        result: list[list[int]] = [[] for _ in prompts]
        for step, gave in zip(tokens, who):
            for b in gave:
                result[b].append(step[b])
        return result


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=8)
    ap.add_argument("--requests", type=int, default=16)
    ap.add_argument("--prompt-tokens", type=int, default=1024)
    ap.add_argument("--new-tokens", type=int, default=64)
    ap.add_argument("--chunk", type=int, default=2048, help="prompt tokens a step")
    ap.add_argument("--page-size", type=int, default=16)
    ap.add_argument("--fp8-qkv", action="store_true", help="e4m3 QKV projection, scales per token")
    args = ap.parse_args(argv)
    shape = DecoderShape(layers=args.layers)
    max_len = args.prompt_tokens + args.new_tokens
    dec = PagedMoEDecoder(shape, max_requests=args.requests, max_len=max_len,
                          max_tokens=args.chunk + args.requests, page_size=args.page_size,
                          fp8_qkv=args.fp8_qkv)
    gen = torch.Generator().manual_seed(0)
    prompts = [torch.randint(shape.vocab, (max(1, args.prompt_tokens - 7 * b),), generator=gen).tolist()
               for b in range(args.requests)]
    times = {}
    for name, n in (("prefill", 1), ("all", args.new_tokens), ("prefill", 1), ("all", args.new_tokens)):
        torch.cuda.synchronize()
        t = time.perf_counter()
        tokens = dec.generate(prompts, n, args.chunk)
        torch.cuda.synchronize()
        times[name] = time.perf_counter() - t
        dec.cache.release(range(args.requests))
    decode = times["all"] - times["prefill"]
    print(json.dumps({
        "workload": f"{args.layers} layers of qwen3-30b-a3b shape, random weights, {args.requests} requests",
        "prompt_tokens": sum(map(len, prompts)), "prefill_s": times["prefill"],
        "prefill_tokens_per_s": sum(map(len, prompts)) / times["prefill"],
        "decode_ms_per_step": 1e3 * decode / max(1, args.new_tokens - 1),
        "fp8_qkv": args.fp8_qkv, "first_tokens": [t[:4] for t in tokens[:2]]}))
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
