"""Tensors that a call would read wrongly are refused: in host memory, or of
strides that are not the call's."""

from __future__ import annotations

import pytest
import torch

from flatrun_amd import device
from test_attention import decode, prefill, rope


def wide(rows, width, dtype=torch.float32):
    return torch.zeros((rows, 2 * width), dtype=dtype)[:, :width]


@pytest.mark.parametrize("call,kw", [
    (rope, dict(x=torch.zeros((3, 1024)))), (rope, dict(table=torch.zeros((16, 64, 2)))),
    (rope, dict(positions=torch.zeros(3, dtype=torch.int32))), (rope, dict(q_norm=torch.zeros(128))),
    (decode, dict(q=torch.zeros((2, 4, 128)))), (decode, dict(lens=torch.zeros(2, dtype=torch.int32))),
    (decode, dict(table=torch.zeros((2, 2), dtype=torch.int32))),
    (prefill, dict(k=torch.zeros((8, 2, 128), dtype=torch.bfloat16))),
    (prefill, dict(cu_q=torch.zeros(2, dtype=torch.int32))),
    (rope, dict(x=wide(3, 1024), ld_x=2048)), (prefill, dict(q=wide(8, 512, torch.bfloat16), ld_q=1024)),
])
def test_host_tensors(call, kw):
    with pytest.raises(ValueError, match="host memory"):
        call(**kw)


@pytest.mark.parametrize("call,kw", [
    (rope, dict(x=wide(3, 1024))), (rope, dict(x=wide(3, 1024), ld_x=1040)), (rope, dict(q=wide(3, 512))),
    (rope, dict(v=torch.zeros((256, 3)).t())), (rope, dict(positions=torch.zeros(6, dtype=torch.int32)[::2])),
    (rope, dict(k_norm=torch.zeros(256)[::2])), (rope, dict(table=torch.zeros((16, 128, 2))[:, :64])),
    (decode, dict(q=wide(2, 512))), (decode, dict(out=torch.zeros((4, 2, 128)).transpose(0, 1))),
    (decode, dict(lens=torch.zeros((2, 2), dtype=torch.int32)[:, 0])),
    (decode, dict(table=torch.zeros((2, 6), dtype=torch.int32)[:, ::3])),
    (prefill, dict(k=torch.zeros((2, 8, 128), dtype=torch.bfloat16).transpose(0, 1))),
    (prefill, dict(v=torch.zeros(8 * 256, dtype=torch.bfloat16)[:1024].view(8, 1, 128).expand(8, 2, 128))),
    (prefill, dict(q=torch.zeros((8, 4, 256), dtype=torch.bfloat16)[..., :128])),
    (prefill, dict(cu_k=torch.zeros((2, 2), dtype=torch.int32)[:, 1])),
])
def test_strides_that_are_not_the_calls(call, kw):
    with pytest.raises(ValueError, match="strides"):
        call(**kw)


@pytest.mark.parametrize("shape,strides,ld,hs,fits", [
    ((3, 1024), (2048, 1), 2048, 0, True), ((3, 8, 128), (2048, 128, 1), 2048, 0, True),
    ((3, 8, 128), (2048, 256, 1), 2048, 0, False), ((3, 8, 128), (2048, 256, 1), 2048, 256, True),
    ((8, 3, 128), (128, 1024, 1), 1024, 128, True), ((2, 3, 512), (1536, 512, 1), 512, 0, True),
    ((2, 5, 512), (5120, 1024, 1), 1024, 0, True), ((2, 5, 512), (6144, 1024, 1), 1024, 0, False),
    ((1, 512), (7, 1), 512, 0, True), ((5, 1), (3, 1), 0, 0, False), ((5, 1), (3, 1), 3, 0, False), ((4, 8), (0, 1), 8, 0, False),
])
def test_rows_of_a_view(shape, strides, ld, hs, fits):
    t = torch.as_strided(torch.zeros(1 << 14), shape, strides)
    assert device._rows_of(t, ld, hs) == fits


def test_no_rows_need_no_bytes():
    """Whatever their strides are."""
    none = torch.zeros((2, 0, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="host memory"):
        prefill(k=none, tokens_k=0, max_k=0, ld_k=128, hs_k=1 << 20)
