"""BlockAttention in DecoderProjections.forward: a prompt, its next chunk and
single tokens through one block, the attention output of each step against
the 64-bit forms on the step's own q|k|v rows."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from attn_ref import attend, block4, rope
from flatrun_amd import device, synth
from flatrun_amd.attention import BlockAttention, KVCache4, Sequence, rope_table
from flatrun_amd.layer import DecoderProjections

pytestmark = pytest.mark.gpu

HQ, HKV, D, HIDDEN, INTER = 8, 2, 64, 512, 768
SPECS = {"q": (HQ * D, HIDDEN), "k": (HKV * D, HIDDEN), "v": (HKV * D, HIDDEN), "o": (HIDDEN, HQ * D),
         "gate": (INTER, HIDDEN), "up": (INTER, HIDDEN), "down": (HIDDEN, INTER)}


def bf16(a):
    return torch.as_tensor(np.asarray(a, np.float32)).bfloat16().double().numpy()


def test_prompts_chunks_and_tokens(frq):
    weights = {p: ("Q4_K", device.DeviceBuffer.from_host(synth.make_blocks("Q4_K", n, k, seed=i)), n, k)
               for i, (p, (n, k)) in enumerate(SPECS.items())}
    table = rope_table(D, 512, base=10000.0)
    rng = np.random.default_rng(0)
    wq, wk = ((1 + 0.2 * rng.standard_normal(D)).astype(np.float32) for _ in range(2))
    cache = KVCache4(16, 32, HKV, D)
    stream = device.Stream()
    step = BlockAttention(cache, HQ, device.DeviceBuffer.from_host(table), 512, max_rows=128, max_seqs=3,
                          max_context=160, q_norm=device.DeviceBuffer.from_host(wq),
                          k_norm=device.DeviceBuffer.from_host(wk), stream=stream)
    seqs = [Sequence() for _ in range(3)]
    held = {s: (np.zeros((0, HKV, D)), np.zeros((0, HKV, D))) for s in seqs}
    with DecoderProjections(weights, max_seq=128, stream=stream) as block:
        # first prompts; the next chunk of one and another prompt; a token each, twice
        for new in ({seqs[0]: 45, seqs[1]: 7}, {seqs[0]: 40, seqs[2]: 33}, {s: 1 for s in seqs}, {s: 1 for s in seqs}):
            rows = sum(new.values())
            start = {s: s.length for s in new}
            step.plan(new)
            x = device.DeviceBuffer.from_host(synth.make_x(rows * HIDDEN, seed=rows))
            block.forward(x, seq=rows, attention=step, post_attention=lambda o, n: o)
            stream.synchronize()
            qkv = block.qkv.to_host(np.float32)[:rows * block.qkv_n].reshape(rows, -1, D)
            got = step.out.to_host(np.float32)[:rows * HQ * D].reshape(rows, HQ, D)
            assert np.isfinite(block.mlp_out.to_host(np.float32)[:rows * HIDDEN]).all()
            single = all(n == 1 for n in new.values())
            context = any(start.values())
            at = 0
            for s, n in new.items():
                assert s.length == start[s] + n and len(s.pages) == -(-s.length // 32)
                pos = np.arange(start[s], s.length)
                (q, k, v), _ = rope(qkv[at:at + n], HQ, HKV, D, D, False, table[pos], wq, wk)
                if not single:
                    q, k, v = bf16(q), bf16(k), bf16(v)
                # a block's code can be one off where its value lies on a tie in 64 bits
                held[s] = tuple(np.concatenate([h, block4(np.float32(a))]) for h, a in zip(held[s], (k, v)))
                kk, vv = held[s] if single or context else (k, v)
                for h in range(HQ):
                    want, mag, _ = attend(q[:, h], kk[:, h // 4], vv[:, h // 4], D ** -0.5, pos)
                    err = np.linalg.norm(got[at:at + n, h] - want) / np.linalg.norm(mag)
                    assert err <= 2e-2, (rows, h, err)
                at += n
    free = cache.take(16 - sum(len(s.pages) for s in seqs))
    assert len(set(free) | {p for s in seqs for p in s.pages}) == 16
    with pytest.raises(Exception):
        cache.take()
    step.close()
    cache.close()
