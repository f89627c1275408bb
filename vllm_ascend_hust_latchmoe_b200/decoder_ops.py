"""The attention half of a decoder layer around the slot-bank MoE layer, on hand-written kernels.

* :func:`add_rms_norm` -- residual addition and RMS norm, bf16 or e4m3 + scales output;
* :func:`build_page_tables`, :func:`release_pages` -- a paged KV cache's block tables, positions
  and slots of one step, from device-side request lengths and a device-side free list;
* :func:`rope_cache_write` -- per-head norm and rotary embedding of a fused QKV output, K and V
  written into the cache;
* :func:`paged_attention` -- attention of single tokens, chunks or prompts over the cache.

Every call takes CUDA tensors that the caller owns (outputs included), launches on the current
stream of the current device, allocates nothing and reads nothing back, so each can be captured in
a CUDA graph. Tensors must live on the current device; one used on another stream than the one it
was written on is ordered by the caller, as for any kernel. Wrong types, shapes or layouts raise
``ValueError``; what only the device can see (a full cache, a bad length) is recorded in
``err_word`` (int32, see ``_lib.DEVERR_NAMES``).
"""

from __future__ import annotations

import ctypes
import importlib.util

import torch

from . import _lib
from ._build import BINDING_PATH, binding_key

_binding = None


def _load():
    """The binding, with the library's entry points: loaded at the first call, and loudly where it
    is missing (there is no other path)."""
    global _binding
    if not BINDING_PATH.exists():
        raise RuntimeError(
            f"{BINDING_PATH.name} is not built at {BINDING_PATH}; run "
            "`python -c 'import __graft_entry__ as g; g.build()'`")
    spec = importlib.util.spec_from_file_location("_decoder_ops", BINDING_PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    if module.built_for != binding_key():
        raise RuntimeError(f"{BINDING_PATH} was built for {module.built_for}, this is {binding_key()}: "
                           "build it again")
    lib = _lib.lib()
    for name in ("lm_last_error", "lm_add_rms_norm", "lm_build_page_tables", "lm_release_pages",
                 "lm_rope_cache_write", "lm_paged_attention"):
        module.bind(name, ctypes.cast(getattr(lib, name), ctypes.c_void_p).value)
    _binding = module
    return module


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *,
                 residual: torch.Tensor | None = None,
                 residual_out: torch.Tensor | None = None,
                 out: torch.Tensor | None = None, out_fp8: torch.Tensor | None = None,
                 scales: torch.Tensor | None = None, group_size: int = 0) -> None:
    """``z = x + residual``; ``residual_out = bf16(z)``;
    ``y = z * rsqrt(mean(z^2) + eps) * weight`` into ``out`` (bf16 ``[T, H]``) or ``out_fp8``
    (e4m3 ``[T, H]``) with fp32 ``scales`` ``[T, 1]`` (``group_size`` 0) or
    ``[T, H / group_size]``: ``scale = max(max|y|, 1e-12) / 448``, ``out_fp8 = e4m3(y / scale)`` (the
    fp32 quotient within 3 units of its last place).

    ``x`` ``[T, H]`` and the other rows may have any row stride; ``residual_out`` may be
    ``residual`` or ``x`` (in place). ``H`` is at most 16384."""
    (_binding or _load()).add_rms_norm(x, weight, eps, residual, residual_out, out, out_fp8, scales,
                                       group_size)


def build_page_tables(cached_lens: torch.Tensor, new_lens: torch.Tensor, page_size: int,
                      block_tables: torch.Tensor, free_pages: torch.Tensor,
                      free_count: torch.Tensor, *, seq_lens: torch.Tensor, cu_q: torch.Tensor,
                      positions: torch.Tensor, slot_mapping: torch.Tensor,
                      free_count_out: torch.Tensor | None = None,
                      err_word: torch.Tensor | None = None) -> None:
    """One step's tables of ``B`` requests from int32 ``cached_lens`` and ``new_lens`` ``[B]``.

    Pages for the new tokens come off the end of the free stack (``free_pages[:free_count]``) in
    request order and go into ``block_tables`` ``[B, max_pages]`` behind the pages held. Writes
    ``seq_lens`` ``[B]``, ``cu_q`` ``[B + 1]``, int32 ``positions`` and int64 ``slot_mapping``
    (as long as the step may have tokens; past the last token position 0 and slot -1) and
    ``free_count_out`` ``[1]`` (``free_count`` itself by default). ``seq_lens`` may be
    ``cached_lens``. A request that finds no page keeps its length and its tokens get slot -1
    (device error 5)."""
    (_binding or _load()).build_page_tables(
        cached_lens, new_lens, page_size, block_tables, free_pages, free_count, seq_lens, cu_q,
        positions, slot_mapping, free_count_out, err_word)


def release_pages(rows: torch.Tensor, cached_lens: torch.Tensor, page_size: int,
                  block_tables: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
                  err_word: torch.Tensor | None = None) -> None:
    """Give the pages of the requests in ``rows`` (int32) back: they go onto the free stack, their
    table entries become -1 and their ``cached_lens`` 0. Entries below 0 (pages that were given back
    before, as behind a sliding window) are passed over."""
    (_binding or _load()).release_pages(rows, cached_lens, page_size, block_tables, free_pages,
                                        free_count, err_word)


def rope_cache_write(qkv: torch.Tensor, positions: torch.Tensor, slot_mapping: torch.Tensor,
                     cos_sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                     q_out: torch.Tensor, *, q_norm_weight: torch.Tensor | None = None,
                     k_norm_weight: torch.Tensor | None = None, eps: float = 1e-6,
                     interleaved: bool = False, err_word: torch.Tensor | None = None) -> None:
    """``qkv`` ``[T, (Hq + 2 Hkv) * D]``: RMS norm over ``D`` of the q and k heads (where weights
    ``[D]`` are given), rotary embedding of their first ``rot_dim`` values, q into ``q_out``
    ``[T, Hq, D]``, k and v into slot ``slot_mapping[t]`` of the caches
    ``[pages, page_size, Hkv, D]`` (slot -1: nowhere). ``cos_sin`` fp32
    ``[max_positions, rot_dim]`` holds the cosines, then the sines; pairs are ``(i, i + rot_dim/2)``
    or neighbours (``interleaved``). ``q_out`` may be a view of ``qkv``'s q part."""
    (_binding or _load()).rope_cache_write(
        qkv, positions, slot_mapping, cos_sin, k_cache, v_cache, q_out, q_norm_weight,
        k_norm_weight, eps, interleaved, err_word)


def attention_workspace(device: torch.device | str | None = None) -> torch.Tensor:
    """A workspace for :func:`paged_attention`, of one size for every call. Calls that share one
    must not overlap (one per stream)."""
    device = torch.device("cuda" if device is None else device)
    with torch.cuda.device(device):
        n = int(_lib.lib().lm_paged_attention_workspace_bytes())
    return torch.zeros(n, dtype=torch.uint8, device=device)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_tables: torch.Tensor, seq_lens: torch.Tensor, cu_q: torch.Tensor,
                    out: torch.Tensor, *, max_q_len: int, workspace: torch.Tensor,
                    scale: float | None = None, window: int = 0,
                    lse: torch.Tensor | None = None,
                    err_word: torch.Tensor | None = None) -> None:
    """Attention of ``q`` ``[T, Hq, D]`` over the paged caches ``[pages, page_size, Hkv, D]`` into
    ``out`` ``[T, Hq, D]`` (and fp32 ``lse`` ``[T, Hq]``).

    Request ``b`` owns tokens ``cu_q[b] .. cu_q[b + 1]``, the last of which stands at position
    ``seq_lens[b] - 1``; a token sees the keys up to its own position, with ``window`` > 0 only the
    last ``window`` of them. A token that sees none gets zeros and an lse of -inf. ``scale``
    defaults to ``D ** -0.5``. ``max_q_len`` (the longest query, as far as the host knows) chooses
    the kernels; the result does not depend on it."""
    (_binding or _load()).paged_attention(
        q, k_cache, v_cache, block_tables, seq_lens, cu_q, out, max_q_len, workspace, scale, window,
        lse, err_word)
