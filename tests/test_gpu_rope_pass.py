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
