"""Argument checks of the decoder operators that need no GPU: they come before any launch."""

import ctypes

import pytest
import torch

from vllm_ascend_hust_latchmoe_b200 import _lib
from vllm_ascend_hust_latchmoe_b200 import decoder_ops as ops

FAKE = ctypes.c_void_p(0x1000)


def _refused(rc, word):
    assert rc < 0 and word in _lib.load().lm_last_error(), (rc, _lib.load().lm_last_error())


def test_norm_arguments_are_checked_on_the_host():
    f = _lib.load().lm_add_rms_norm

    def call(H=64, T=2, stride=64, x=FAKE, y=FAKE, y8=None, scales=None, group=0):
        return f(x, stride, None, 0, FAKE, 1e-6, T, H, None, 0, y, stride, y8, stride, scales, group, None)

    assert call(T=0) == 0  # nothing to do, no CUDA call
    _refused(call(H=0), b"hidden_size")
    _refused(call(H=16385, stride=20000), b"hidden_size")
    _refused(call(T=-1), b"num_tokens")
    _refused(call(stride=63), b"stride")
    _refused(call(x=None), b"null")
    _refused(call(y=None), b"one of y and y8")
    _refused(call(y8=FAKE, scales=FAKE), b"one of y and y8")
    _refused(call(y=None, y8=FAKE), b"scales")
    _refused(call(y=None, y8=FAKE, scales=FAKE, group=40), b"group_size")


def test_table_arguments_are_checked_on_the_host():
    f = _lib.load().lm_build_page_tables

    def call(B=2, page=16, width=4, stride=4, T=8, cached=FAKE, count=FAKE):
        return f(cached, FAKE, B, page, FAKE, stride, width, FAKE, 8, count, FAKE, FAKE, FAKE, FAKE, FAKE, T,
                 None, None)

    for kw in (dict(page=0), dict(width=0), dict(stride=3), dict(T=-1), dict(width=1 << 28, stride=1 << 28)):
        _refused(call(**kw), b"bad sizes")
    _refused(call(B=4097), b"4096")
    _refused(call(cached=None), b"null")
    _refused(call(count=None), b"null")
    r = _lib.load().lm_release_pages
    assert r(None, 0, FAKE, 2, 16, FAKE, 4, 4, FAKE, 8, FAKE, None, None) == 0
    _refused(r(FAKE, 1, FAKE, 0, 16, FAKE, 4, 4, FAKE, 8, FAKE, None, None), b"bad sizes")
    _refused(r(None, 1, FAKE, 2, 16, FAKE, 4, 4, FAKE, 8, FAKE, None, None), b"null")


def test_rope_arguments_are_checked_on_the_host():
    f = _lib.load().lm_rope_cache_write

    def call(D=64, R=64, T=1, heads=4, qkv=FAKE, page=16, stride=8 * 64):
        return f(qkv, stride, FAKE, FAKE, T, heads, 2, D, FAKE, 16, R, 0, None, None, 1e-6, FAKE, 256, 64, FAKE,
                 2048, 128, 64, FAKE, 2048, 128, 64, 4, page, None, None)

    assert call(T=0) == 0
    _refused(call(D=96), b"head_dim")
    _refused(call(R=66), b"rot_dim")
    _refused(call(R=33), b"rot_dim")
    _refused(call(heads=0), b"bad sizes")
    _refused(call(page=0), b"bad sizes")
    _refused(call(qkv=None), b"null")
    _refused(call(qkv=ctypes.c_void_p(0x1002)), b"16-byte")
    _refused(call(stride=8 * 64 + 1), b"multiples of 8")


def test_attention_arguments_are_checked_on_the_host():
    lib = _lib.load()

    def call(D=64, Hq=4, Hkv=2, page=16, B=1, T=1, window=0, q=FAKE, stride=64, ws=1 << 40, width=4):
        return lib.lm_paged_attention(q, 256, stride, FAKE, 2048, 128, 64, FAKE, 2048, 128, 64, 4, page, FAKE,
                                      width, width, FAKE, FAKE, B, T, Hq, Hkv, D, 1, 0.125, window, FAKE, 256, 64,
                                      None, FAKE, ws, None, None)

    assert call(B=0) == 0 and call(T=0) == 0
    _refused(call(D=96), b"head_dim")
    _refused(call(Hq=5), b"multiple of num_kv_heads")
    _refused(call(page=8), b"page_size")
    _refused(call(B=4097), b"4096")
    _refused(call(window=-1), b"bad sizes")
    _refused(call(width=0), b"bad sizes")
    _refused(call(q=None), b"null")
    _refused(call(q=ctypes.c_void_p(0x1004)), b"16-byte")
    _refused(call(stride=60), b"multiples of 8")
    _refused(call(ws=64), b"workspace")


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.add_rms_norm(x, x[0], out=x)
    kc = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention(x.view(2, 1, 64), kc, kc, torch.zeros(1, 2), torch.zeros(1), torch.zeros(2),
                            x.view(2, 1, 64), max_q_len=1, workspace=torch.zeros(1))


def test_sizes_past_the_counters_are_refused():
    lib = _lib.load()
    rc = lib.lm_add_rms_norm(FAKE, 64, None, 0, FAKE, 1e-6, 1 << 30, 64, None, 0, FAKE, 64, None, 64, None, 0, None)
    _refused(rc, b"2^30")
    # 2^22 single-token requests' rows over 2^24-token rows of the block table: more units than 32 bits count
    rc = lib.lm_paged_attention(FAKE, 256, 64, FAKE, 2048, 128, 64, FAKE, 2048, 128, 64, 4, 16, FAKE, 1 << 20,
                                1 << 20, FAKE, FAKE, 1, 1 << 24, 4, 2, 64, 1, 0.125, 0, FAKE, 256, 64, None, FAKE,
                                1 << 40, None, None)
    _refused(rc, b"too much work")
