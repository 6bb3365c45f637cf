"""Elements that qk_norm_rope does not turn pass as they are, whatever stands
beside them: an inf or a NaN reaches its own pair at most."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from attn_ref import dev
from flatrun_amd import device
from flatrun_amd.attention import rope_table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 80, 128, 256])
@pytest.mark.parametrize("part", [0, 8, 4])                        # of the head that turns: none, an eighth, a quarter
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_elements_past_the_turned_part(frq, d, part, inter, bad):
    rot = d // part // 4 * 4 if part else 0
    g = torch.Generator().manual_seed(d)
    x = torch.randn((5, 3, d), generator=g)
    x[1, 0, d - 1], x[2, 1, rot + 2], x[3, 0, d // 2 + 3] = bad, bad, bad
    out = [torch.zeros((5, 1, d), device="cuda") for _ in range(3)]
    device.qk_norm_rope(x.cuda(), *out, 5, 1, 1, d, dev(rope_table(max(rot, 2), 16)), dev(np.arange(5, dtype=np.int32)),
                        rot=rot, interleaved=inter)
    torch.cuda.synchronize()
    for i in range(3):
        got = out[i].cpu()[:, 0]
        lo = rot if i < 2 else 0
        assert torch.equal(torch.nan_to_num(got[:, lo:], nan=7e7), torch.nan_to_num(x[:, i, lo:], nan=7e7))
        assert torch.isfinite(got[:, :lo]).all()


def test_more_tokens_than_one_launch_takes(frq):
    """2^24 workgroups of 256 threads are one too many."""
    n, d = (1 << 24) + 3, 8
    row = torch.randn((1 << 12, 2 * d)).bfloat16()
    x = row.cuda().repeat((n >> 12) + 1, 1)[:n].contiguous()
    q, k = (torch.zeros((n, d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table, pos = dev(rope_table(d, 4096)), torch.arange(n, dtype=torch.int32, device="cuda") % 4096
    device.qk_norm_rope(x, q, k, None, n, 1, 1, d, table, pos, x_dtype="bf16", out_dtype="bf16")
    torch.cuda.synchronize()
    for t in (q, k):
        assert torch.isfinite(t[:4096]).all() and t[:4096].abs().sum() > 0
        assert torch.equal(t[:n >> 12 << 12].view(-1, 4096, d), t[:4096].expand(n >> 12, 4096, d))
        assert torch.equal(t[n >> 12 << 12:], t[:3])
