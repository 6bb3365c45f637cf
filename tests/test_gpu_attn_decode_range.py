"""attn_decode where sizes differ inside a head: blocks of channels, single
tokens, queries, and weights far below the largest. The bound is the one of
test_gpu_attn_decode (attn_ref.fp32_bound), channel by channel."""

from __future__ import annotations

import numpy as np
import pytest

from attn_ref import block4, dev
from test_gpu_attn_decode import Setup

pytestmark = pytest.mark.gpu


def write(s):
    s.cache.write(dev(s.k), dev(s.v), dev(s.slots), sum(s.lens))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("small", [2.0 ** -8, 1e-3, 1e-5, 1e-6])
@pytest.mark.parametrize("block", [0, 1])
def test_blocks_of_v_of_different_size(frq, d, small, block):
    s = Setup([311, 33, 1], 4, 2, d, 32, seed=21, spare=0)
    s.v[:, 1, 32 * block:32 * block + 32] *= small
    s.v[:, 0, d - 32:] /= small                              # up to the largest scale that a block takes
    s.v = np.clip(s.v, -5e5, 5e5)
    write(s)
    s.check(s.run())


@pytest.mark.parametrize("n,page", [(300, 32), (4000, 64)])
def test_a_token_of_large_values_and_no_weight(frq, n, page):
    """In the first tile, in a later one and in the last."""
    for at in (0, n // 2, n - 1):
        s = Setup([n], 8, 2, 128, page, seed=22, spare=0)
        s.k[at] = -40 * np.sign(s.q.numpy().reshape(1, 2, 4, 128).sum(2)[0])      # scores far below the others
        s.v[at] *= 4096
        write(s)
        s.check(s.run())


@pytest.mark.parametrize("d,n", [(64, 700), (128, 5000), (256, 300)])
def test_a_token_with_nearly_all_weight_and_no_value(frq, d, n):
    """The others, 2^-24 of its weight, make the output."""
    s = Setup([n], 2, 2, d, 64, seed=23, spare=0)
    q = s.q.numpy()[0]
    s.k *= 0.2
    s.k[0] = q * (24 * np.log(2) * d ** 0.5 / (q * q).sum(-1, keepdims=True))
    s.v[0] = 0
    write(s)
    s.check(s.run())


def test_queries_whose_blocks_differ_as_the_keys_do(frq):
    s = Setup([200, 40], 4, 2, 64, 32, seed=24, spare=0)
    s.q[..., :32] *= 2.0 ** -28
    s.k[..., :32] *= 2.0 ** 14
    s.k[..., 32:] *= 2.0 ** -14
    s.q *= 2.0 ** 14
    write(s)
    s.check(s.run())


def test_same_bits_every_time(frq):
    s = Setup([2500, 7, 0, 900], 8, 2, 128, 64, seed=25)
    s.v[..., :32] *= 1e-4
    write(s)
    assert np.array_equal(s.run(), s.run())


@pytest.mark.parametrize("n,low", [(100, 40), (100, 99), (5000, 700), (5000, 4999)])
def test_tokens_whose_scores_overflow(frq, n, low):
    """-inf in fp32: no weight, wherever it stands, as the definition has it; NaN where nothing else is left."""
    s = Setup([n, 20], 8, 2, 64, 32, seed=26, spare=0)
    s.q[0] = 0
    s.q[0, :, 0] = 3e38
    s.k[:n, :, :32] = 0
    s.k[:low, :, 0] = -1000.0
    write(s)
    got = s.run()
    v = block4(s.v[low:n]).repeat(4, axis=1)                 # equal weights of the others
    assert np.all(np.abs(got[0] - v.mean(0)) <= (2.0 ** -20 + 8 * n ** 0.5 * 2.0 ** -24) * np.abs(v).mean(0))
    s.k[:n, :, 0] = -1000.0
    write(s)
    assert np.isnan(s.run()[0]).all() and np.array_equal(s.run()[1], got[1])
