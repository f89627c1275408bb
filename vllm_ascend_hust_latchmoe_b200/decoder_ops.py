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

import torch

from . import _lib

_BF16 = torch.bfloat16
_I32 = torch.int32
_F32 = torch.float32


_I64 = torch.int64
_E4M3 = torch.float8_e4m3fn

# The calls are short next to a launch, so their checks are too: one expression of plain
# comparisons over everything, and the function that says what is wrong only where it fails
# (5 us of a 16-token norm's 7 us of host time otherwise, and 3 us more through
# torch.cuda.current_stream).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _stream(device: int) -> int:
    """The current stream of the tensors' device, which has to be the current one: the library
    launches there."""
    if _current_device() != device:
        raise ValueError(f"the tensors are on cuda:{device}, which is not the current device")
    if _raw_stream is not None:
        return _raw_stream(device)
    return torch.cuda.current_stream(device).cuda_stream


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _check_tensor(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple) -> None:
    """dtype, device and shape of one argument (None in ``shape``: any size)."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    got = t.shape
    if len(got) != len(shape) or any(w is not None and w != g for w, g in zip(shape, got)):
        raise ValueError(f"{name} must have shape {shape}, not {tuple(got)}")


def _check_dense(name: str, t: torch.Tensor) -> None:
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _check_device(*tensors: torch.Tensor | None) -> None:
    devices = {t.device for t in tensors if t is not None}
    if len(devices) > 1:
        raise ValueError(f"the tensors are on several devices: {sorted(map(str, devices))}")


def _check_err(err_word: torch.Tensor | None, device: int) -> int | None:
    if err_word is None:
        return None
    _check_tensor("err_word", err_word, _I32, (1,))
    _need(err_word.get_device() == device, "err_word is on another device")
    return err_word.data_ptr()


def _vector(t: torch.Tensor, dtype: torch.dtype, n: int, device: int) -> bool:
    return (t.dtype is dtype and t.shape == (n,) and t.get_device() == device and t.is_contiguous())


def _rows(t: torch.Tensor, dtype: torch.dtype, shape: torch.Size, device: int) -> bool:
    """Contiguous rows that do not overlap (other layouts take the slow check)."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device:
        return False
    stride = t.stride()
    return stride[1] == 1 and stride[0] >= shape[1]


def _row_stride(t: torch.Tensor) -> int:
    """Row stride in elements; of a single row, what a dense layout has."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[-1])


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *,
                 residual: torch.Tensor | None = None,
                 residual_out: torch.Tensor | None = None,
                 out: torch.Tensor | None = None, out_fp8: torch.Tensor | None = None,
                 scales: torch.Tensor | None = None, group_size: int = 0) -> None:
    """``z = x + residual``; ``residual_out = bf16(z)``;
    ``y = z * rsqrt(mean(z^2) + eps) * weight`` into ``out`` (bf16 ``[T, H]``) or ``out_fp8``
    (e4m3 ``[T, H]``) with fp32 ``scales`` ``[T, 1]`` (``group_size`` 0) or
    ``[T, H / group_size]``: ``scale = max(max|y|, 1e-12) / 448``, ``out_fp8 = e4m3(y / scale)``.

    ``x`` ``[T, H]`` and the other rows may have any row stride; ``residual_out`` may be
    ``residual`` or ``x`` (in place). ``H`` is at most 16384."""
    y, y_dtype = (out, _BF16) if out is not None else (out_fp8, _E4M3)
    dev, shape = x.get_device(), x.shape
    good = (dev >= 0 and len(shape) == 2 and _rows(x, _BF16, shape, dev) and y is not None
            and _rows(y, y_dtype, shape, dev) and _vector(weight, _BF16, shape[1], dev)
            and (residual is None or _rows(residual, _BF16, shape, dev))
            and (residual_out is None or _rows(residual_out, _BF16, shape, dev))
            and (scales is None and group_size == 0 if out_fp8 is None else
                 out is None and scales is not None and scales.dtype is _F32
                 and (group_size == 0 or (group_size % 32 == 0 and shape[1] % group_size == 0))
                 and scales.shape == (shape[0], shape[1] // group_size if group_size else 1)
                 and scales.get_device() == dev and scales.is_contiguous()))
    if not good:
        _check_norm(x, weight, residual, residual_out, out, out_fp8, scales, group_size)
    T, H = shape
    y_ptr, y_stride = y.data_ptr(), _row_stride(y)
    rc = _lib.lib().lm_add_rms_norm(
        x.data_ptr(), _row_stride(x), _ptr(residual),
        0 if residual is None else _row_stride(residual), weight.data_ptr(), eps, T, H,
        _ptr(residual_out), 0 if residual_out is None else _row_stride(residual_out),
        None if out is None else y_ptr, y_stride, None if out_fp8 is None else y_ptr, y_stride,
        _ptr(scales), group_size, _stream(dev))
    if rc < 0:
        _lib._check("lm_add_rms_norm", rc)


def _check_norm(x, weight, residual, residual_out, out, out_fp8, scales, group_size) -> None:
    _need(x.dim() == 2, "x must be [tokens, hidden]")
    T, H = x.shape
    _check_tensor("x", x, _BF16, (T, H))
    _check_tensor("weight", weight, _BF16, (H,))
    _check_dense("weight", weight)
    _need((out is None) != (out_fp8 is None), "give one of out and out_fp8")
    y, y_dtype = (out, _BF16) if out is not None else (out_fp8, torch.float8_e4m3fn)
    _check_tensor("out", y, y_dtype, (T, H))
    rows = [("x", x), ("out", y)]
    if residual is not None:
        _check_tensor("residual", residual, _BF16, (T, H))
        rows.append(("residual", residual))
    if residual_out is not None:
        _check_tensor("residual_out", residual_out, _BF16, (T, H))
        rows.append(("residual_out", residual_out))
    for name, t in rows:
        _need(H <= 1 or t.stride(1) == 1, f"{name}'s rows must be contiguous")
        _need(T <= 1 or t.stride(0) >= H, f"{name}'s rows overlap")
    if out_fp8 is not None:
        _need(group_size >= 0 and (group_size == 0 or (group_size % 32 == 0 and H % group_size == 0)),
              "group_size must be 0 or a multiple of 32 that divides the hidden size")
        _need(scales is not None, "out_fp8 needs scales")
        _check_tensor("scales", scales, _F32, (T, H // group_size if group_size else 1))
        _check_dense("scales", scales)
    else:
        _need(scales is None and not group_size, "scales belong to out_fp8")
    _check_device(x, weight, residual, residual_out, out, out_fp8, scales)


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
    if free_count_out is None:
        free_count_out = free_count
    dev, B, T = cached_lens.get_device(), cached_lens.numel(), positions.numel()
    good = (dev >= 0 and block_tables.dtype is _I32 and block_tables.dim() == 2
            and block_tables.shape[0] == B and block_tables.shape[1] > 0
            and block_tables.get_device() == dev and block_tables.stride(1) == 1
            and _vector(cached_lens, _I32, B, dev) and _vector(new_lens, _I32, B, dev)
            and _vector(free_pages, _I32, free_pages.numel(), dev)
            and _vector(free_count, _I32, 1, dev) and _vector(free_count_out, _I32, 1, dev)
            and _vector(seq_lens, _I32, B, dev) and _vector(cu_q, _I32, B + 1, dev)
            and _vector(positions, _I32, T, dev) and _vector(slot_mapping, _I64, T, dev))
    if not good:
        _check_tables(cached_lens, new_lens, block_tables, free_pages, free_count, free_count_out,
                      seq_lens, cu_q, positions, slot_mapping)
    width = block_tables.shape[1]
    rc = _lib.lib().lm_build_page_tables(
        cached_lens.data_ptr(), new_lens.data_ptr(), B, page_size, block_tables.data_ptr(),
        _row_stride(block_tables) if B else width, width, free_pages.data_ptr(),
        free_pages.shape[0], free_count.data_ptr(), free_count_out.data_ptr(),
        seq_lens.data_ptr(), cu_q.data_ptr(), positions.data_ptr(), slot_mapping.data_ptr(), T,
        _check_err(err_word, dev), _stream(dev))
    if rc < 0:
        _lib._check("lm_build_page_tables", rc)


def _check_tables(cached_lens, new_lens, block_tables, free_pages, free_count, free_count_out,
                  seq_lens, cu_q, positions, slot_mapping) -> None:
    _need(cached_lens.dim() == 1 and block_tables.dim() == 2 and free_pages.dim() == 1
          and positions.dim() == 1, "lengths, free_pages and positions are vectors, block_tables a matrix")
    B, T = cached_lens.shape[0], positions.shape[0]
    for name, t, dtype, shape in (
            ("cached_lens", cached_lens, _I32, (B,)), ("new_lens", new_lens, _I32, (B,)),
            ("free_pages", free_pages, _I32, (None,)), ("free_count", free_count, _I32, (1,)),
            ("free_count_out", free_count_out, _I32, (1,)), ("seq_lens", seq_lens, _I32, (B,)),
            ("cu_q", cu_q, _I32, (B + 1,)), ("positions", positions, _I32, (T,)),
            ("slot_mapping", slot_mapping, torch.int64, (T,))):
        _check_tensor(name, t, dtype, shape)
        _check_dense(name, t)
    _check_tensor("block_tables", block_tables, _I32, (B, None))
    width = block_tables.shape[1]
    _need(width > 0 and (width == 1 or block_tables.stride(1) == 1),
          "block_tables' rows must be contiguous and not empty")
    _check_device(cached_lens, new_lens, block_tables, free_pages, free_count, free_count_out,
                  seq_lens, cu_q, positions, slot_mapping)


def release_pages(rows: torch.Tensor, cached_lens: torch.Tensor, page_size: int,
                  block_tables: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
                  err_word: torch.Tensor | None = None) -> None:
    """Give the pages of the requests in ``rows`` (int32) back: they go onto the free stack, their
    table entries become -1 and their ``cached_lens`` 0."""
    _need(rows.dim() == 1 and block_tables.dim() == 2, "rows is a vector, block_tables a matrix")
    B = block_tables.shape[0]
    for name, t, shape in (("rows", rows, (None,)), ("cached_lens", cached_lens, (B,)),
                           ("free_pages", free_pages, (None,)), ("free_count", free_count, (1,))):
        _check_tensor(name, t, _I32, shape)
        _check_dense(name, t)
    _check_tensor("block_tables", block_tables, _I32, (B, None))
    width = block_tables.shape[1]
    _need(width > 0 and (width == 1 or block_tables.stride(1) == 1),
          "block_tables' rows must be contiguous and not empty")
    _check_device(rows, cached_lens, block_tables, free_pages, free_count)
    dev = rows.get_device()
    _lib._check("lm_release_pages", _lib.lib().lm_release_pages(
        rows.data_ptr(), rows.shape[0], cached_lens.data_ptr(), B, page_size,
        block_tables.data_ptr(), _row_stride(block_tables), width, free_pages.data_ptr(),
        free_pages.shape[0], free_count.data_ptr(), _check_err(err_word, dev), _stream(dev)))


def _check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor) -> tuple:
    _need(k_cache.dim() == 4, "k_cache must be [pages, page_size, kv_heads, head_dim]")
    shape = tuple(k_cache.shape)
    _check_tensor("k_cache", k_cache, _BF16, shape)
    _check_tensor("v_cache", v_cache, _BF16, shape)
    _need(k_cache.stride(3) == 1 and v_cache.stride(3) == 1, "the cache's heads must be contiguous")
    return shape


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
    dev, cache, ks, vs, qs = (k_cache.get_device(), k_cache.shape, k_cache.stride(),
                              v_cache.stride(), q_out.stride())
    good = (dev >= 0 and len(cache) == 4 and len(qs) == 3 and k_cache.dtype is _BF16
            and v_cache.dtype is _BF16 and v_cache.shape == cache and v_cache.get_device() == dev
            and ks[3] == 1 and vs[3] == 1 and qs[2] == 1 and q_out.dtype is _BF16
            and q_out.get_device() == dev and q_out.shape[2] == cache[3] and q_out.shape[0] > 0
            and qkv.dtype is _BF16 and qkv.get_device() == dev and qkv.stride(-1) == 1
            and qkv.shape == (q_out.shape[0], (q_out.shape[1] + 2 * cache[2]) * cache[3])
            and _vector(positions, _I32, q_out.shape[0], dev)
            and _vector(slot_mapping, _I64, q_out.shape[0], dev)
            and cos_sin.dtype is _F32 and cos_sin.dim() == 2 and cos_sin.get_device() == dev
            and cos_sin.is_contiguous()
            and (q_norm_weight is None or _vector(q_norm_weight, _BF16, cache[3], dev))
            and (k_norm_weight is None or _vector(k_norm_weight, _BF16, cache[3], dev)))
    if not good:
        _check_rope(qkv, positions, slot_mapping, cos_sin, k_cache, v_cache, q_out, q_norm_weight,
                    k_norm_weight)
    T, Hq, D = q_out.shape
    rc = _lib.lib().lm_rope_cache_write(
        qkv.data_ptr(), _row_stride(qkv) if T else 0, positions.data_ptr(),
        slot_mapping.data_ptr(), T, Hq, cache[2], D, cos_sin.data_ptr(), cos_sin.shape[0],
        cos_sin.shape[1], 1 if interleaved else 0, _ptr(q_norm_weight), _ptr(k_norm_weight), eps,
        q_out.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), ks[0], ks[1], ks[2],
        v_cache.data_ptr(), vs[0], vs[1], vs[2], cache[0], cache[1], _check_err(err_word, dev),
        _stream(dev))
    if rc < 0:
        _lib._check("lm_rope_cache_write", rc)


def _check_rope(qkv, positions, slot_mapping, cos_sin, k_cache, v_cache, q_out, q_norm_weight,
                k_norm_weight) -> None:
    pages, page_size, Hkv, D = _check_cache(k_cache, v_cache)
    _need(qkv.dim() == 2 and q_out.dim() == 3 and cos_sin.dim() == 2,
          "qkv and cos_sin are matrices, q_out is [tokens, heads, head_dim]")
    T, Hq = q_out.shape[0], q_out.shape[1]
    _check_tensor("qkv", qkv, _BF16, (T, (Hq + 2 * Hkv) * D))
    _check_tensor("q_out", q_out, _BF16, (T, Hq, D))
    _check_tensor("positions", positions, _I32, (T,))
    _check_tensor("slot_mapping", slot_mapping, torch.int64, (T,))
    _check_tensor("cos_sin", cos_sin, _F32, (None, None))
    for name, t in (("positions", positions), ("slot_mapping", slot_mapping), ("cos_sin", cos_sin)):
        _check_dense(name, t)
    for name, t in (("q_norm_weight", q_norm_weight), ("k_norm_weight", k_norm_weight)):
        if t is not None:
            _check_tensor(name, t, _BF16, (D,))
            _check_dense(name, t)
    _need(T == 0 or (qkv.stride(1) == 1 and q_out.stride(2) == 1), "rows and heads must be contiguous")
    _check_device(qkv, positions, slot_mapping, cos_sin, k_cache, v_cache, q_out, q_norm_weight,
                  k_norm_weight)


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
    dev, cache, shape = q.get_device(), k_cache.shape, q.shape
    ks, vs, qs, os = k_cache.stride(), v_cache.stride(), q.stride(), out.stride()
    B = block_tables.shape[0] if block_tables.dim() == 2 else -1
    good = (dev >= 0 and len(cache) == 4 and len(shape) == 3 and k_cache.dtype is _BF16
            and v_cache.dtype is _BF16 and v_cache.shape == cache and k_cache.get_device() == dev
            and v_cache.get_device() == dev and ks[3] == 1 and vs[3] == 1
            and q.dtype is _BF16 and shape[2] == cache[3] and qs[2] == 1 and shape[0] > 0
            and out.dtype is _BF16 and out.shape == shape and os[2] == 1
            and out.get_device() == dev and block_tables.dtype is _I32 and block_tables.dim() == 2
            and block_tables.get_device() == dev and block_tables.stride(1) == 1
            and block_tables.shape[1] > 0 and _vector(seq_lens, _I32, B, dev)
            and _vector(cu_q, _I32, B + 1, dev) and workspace.dtype is torch.uint8
            and workspace.get_device() == dev and workspace.dim() == 1
            and (lse is None or (lse.dtype is _F32 and lse.shape == shape[:2]
                                 and lse.get_device() == dev and lse.is_contiguous())))
    if not good:
        _check_attention(q, k_cache, v_cache, block_tables, seq_lens, cu_q, out, workspace, lse)
    T, Hq, D = shape
    width = block_tables.shape[1]
    rc = _lib.lib().lm_paged_attention(
        q.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), ks[0], ks[1], ks[2], v_cache.data_ptr(),
        vs[0], vs[1], vs[2], cache[0], cache[1], block_tables.data_ptr(),
        _row_stride(block_tables) if B else width, width, seq_lens.data_ptr(), cu_q.data_ptr(), B,
        T, Hq, cache[2], D, max_q_len, D ** -0.5 if scale is None else scale, window,
        out.data_ptr(), os[0], os[1], _ptr(lse), workspace.data_ptr(), workspace.numel(),
        _check_err(err_word, dev), _stream(dev))
    if rc < 0:
        _lib._check("lm_paged_attention", rc)


def _check_attention(q, k_cache, v_cache, block_tables, seq_lens, cu_q, out, workspace,
                     lse) -> None:
    pages, page_size, Hkv, D = _check_cache(k_cache, v_cache)
    _need(q.dim() == 3 and block_tables.dim() == 2, "q is [tokens, heads, head_dim], block_tables a matrix")
    T, Hq = q.shape[0], q.shape[1]
    B, width = block_tables.shape
    _check_tensor("q", q, _BF16, (T, Hq, D))
    _check_tensor("out", out, _BF16, (T, Hq, D))
    _check_tensor("block_tables", block_tables, _I32, (B, width))
    _check_tensor("seq_lens", seq_lens, _I32, (B,))
    _check_tensor("cu_q", cu_q, _I32, (B + 1,))
    _check_tensor("workspace", workspace, torch.uint8, (None,))
    _need(T == 0 or (q.stride(2) == 1 and out.stride(2) == 1), "heads must be contiguous")
    _need(width > 0 and (width == 1 or block_tables.stride(1) == 1),
          "block_tables' rows must be contiguous and not empty")
    for name, t in (("seq_lens", seq_lens), ("cu_q", cu_q), ("workspace", workspace)):
        _check_dense(name, t)
    if lse is not None:
        _check_tensor("lse", lse, _F32, (T, Hq))
        _check_dense("lse", lse)
    _check_device(q, k_cache, v_cache, block_tables, seq_lens, cu_q, out, workspace, lse)
