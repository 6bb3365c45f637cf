"""sample against its definition in 64 bits, with a sort.

Tokens are equal: the kernel's weights are within 2^-45 of the largest of the
64-bit ones, so a sum's border moves by about 2^-45 sqrt(vocab) of the whole
and a draw lands between the two by a chance far below 1e-6. Probabilities are
within that and one rounding to fp32."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from attn_ref import TORCH, dev
from flatrun_amd import device

pytestmark = pytest.mark.gpu


def oracle(x, u, temp, top_k, top_p, min_p):
    """(token, probability, every index that stays) of one row."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if np.all(x == -np.inf):
        return -1, 0.0, np.array([], int)
    if not temp > 0:
        return int(x.argmax()), 1.0, np.array([x.argmax()])
    with np.errstate(invalid="ignore"):
        w = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / temp))
    order = np.lexsort((np.arange(len(x)), -x))
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        upto = np.cumsum(w[order])
        order = order[:1 + np.searchsorted(upto, top_p * upto[-1], side="left")]
    stay = np.sort(order[w[order] >= min(min_p, 1.0)])
    stay = stay[w[stay] > 0]
    upto = np.cumsum(w[stay])
    at = min(int(np.searchsorted(upto, max(u, 0.0) * upto[-1], side="right")), len(stay) - 1)
    return int(stay[at]), w[stay[at]] / upto[-1], stay


def run(x, u, dtype="f32", ld=0, stream=None, **par):
    rows, vocab = u.shape[0], par.pop("vocab", x.shape[-1])
    tok = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    prob = torch.full((rows,), -7.0, device="cuda")
    device.sample(x, dev(u), tok, rows, vocab, probs=prob, dtype=dtype, ld=ld, stream=stream, **par)
    torch.cuda.synchronize()
    return tok.cpu().numpy(), prob.cpu().numpy()


def check(x, u, got, temp, top_k, top_p, min_p):
    """x as the kernel read it (numpy), parameters per row."""
    for i, (t, p) in enumerate(zip(*got)):
        want, share, stay = oracle(x[i], float(u[i]), temp[i], top_k[i], top_p[i], min_p[i])
        assert t == want, (i, t, want, len(stay))
        assert abs(p - share) <= 2.0 ** -23 * share + 1e-9, (i, p, share)


def logits(rows, vocab, seed, dtype="f32", spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn((rows, vocab), generator=g)
    x[:, :: max(1, vocab // 20)] += 6
    return x.to(TORCH[dtype])


def uniform(rows, seed):
    return np.random.default_rng(seed).random(rows, dtype=np.float32)


PARAMS = [dict(), dict(temperature=0.0), dict(temperature=0.3), dict(temperature=1.5, min_p=0.05), dict(top_k=1),
          dict(top_k=40), dict(top_k=1000, temperature=2.0), dict(top_p=0.5), dict(top_p=0.95, temperature=0.75),
          dict(top_p=0.99, temperature=1.5), dict(top_k=50, top_p=0.9), dict(top_k=700, top_p=0.97, min_p=0.01),
          dict(top_p=0.0), dict(min_p=1.0)]


def spelled(rows, par):
    full = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) | par
    return [[float(np.float32(full["temperature"]))] * rows, [full["top_k"]] * rows, [float(np.float32(full["top_p"]))] * rows,
            [float(np.float32(full["min_p"]))] * rows]


@pytest.mark.parametrize("par", PARAMS, ids=[" ".join(f"{k}={v}" for k, v in p.items()) or "free" for p in PARAMS])
@pytest.mark.parametrize("vocab,dtype", [(1000, "f32"), (32003, "bf16"), (50257, "f16"), (152064, "f32")])
def test_parameters(frq, vocab, dtype, par):
    rows = 6
    x, u = logits(rows, vocab, vocab + len(par), dtype), uniform(rows, vocab)
    check(x.float().numpy(), u, run(x.cuda(), u, dtype, **par), *spelled(rows, par))


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 255, 256, 257, 1023, 1025, 4097, 16384, 65537, 262144, 1 << 20])
def test_sizes(frq, vocab):
    rows = 3
    x, u = logits(rows, vocab, vocab), uniform(rows, vocab)
    for par in (dict(), dict(top_k=5, top_p=0.9), dict(top_p=0.8)):
        check(x.numpy(), u, run(x.cuda(), u, **par), *spelled(rows, par))


@pytest.mark.parametrize("rows", [1, 2, 17, 64, 129, 300])
def test_every_row_its_own_parameters(frq, rows):
    vocab = 8191
    x, u = logits(rows, vocab, rows), uniform(rows, rows)
    rng = np.random.default_rng(rows)
    temp = rng.choice(np.array([0, 0.2, 0.7, 1, 1.6], np.float32), rows)
    top_k = rng.choice(np.array([0, 1, 7, 100, 5000, 9000], np.int32), rows)
    top_p = rng.choice(np.array([1, 0.99, 0.9, 0.3], np.float32), rows)
    min_p = rng.choice(np.array([0, 0.01, 0.2], np.float32), rows)
    got = run(x.cuda(), u, temperature=dev(temp), top_k=dev(top_k), top_p=dev(top_p), min_p=dev(min_p))
    check(x.numpy(), u, got, temp.astype(float), top_k, top_p.astype(float), min_p.astype(float))


@pytest.mark.parametrize("par", [dict(), dict(top_k=300), dict(top_p=0.4), dict(top_k=5000, top_p=0.7, min_p=0.5),
                                 dict(temperature=50.0, top_p=0.6), dict(temperature=1e-3, top_k=9, top_p=0.5)])
@pytest.mark.parametrize("kind", ["one value", "two values", "a few values", "dense"])
def test_ties_and_dense_rows(frq, par, kind):
    """Equal logits stay from the lowest index on; more of them in a row than any list holds."""
    rows, vocab = 4, 40000
    rng = np.random.default_rng(len(kind))
    x = {"one value": np.full((rows, vocab), -3.5), "two values": rng.integers(0, 2, (rows, vocab)) * 2.0,
         "a few values": rng.integers(-3, 3, (rows, vocab)) * 0.25,
         "dense": 1 + 1e-4 * rng.standard_normal((rows, vocab))}[kind].astype(np.float32)
    u = uniform(rows, 5)
    check(x, u, run(dev(x), u, **par), *spelled(rows, par))


def test_zeros_of_either_sign_are_equal(frq):
    x = np.where(np.arange(512) % 2, 0.0, -0.0).astype(np.float32)[None].repeat(2, 0)
    u = np.array([0.0, 0.999], np.float32)
    for par in (dict(temperature=0.0), dict(top_k=3), dict(top_p=0.5)):
        check(x, u, run(dev(x), u, **par), *spelled(2, par))


def test_masked_infinite_and_missing_logits(frq):
    """-inf and NaN are never drawn, +inf alone is; a row of nothing gives -1."""
    rows, vocab = 8, 3000
    x = logits(rows, vocab, 3).numpy()
    x[0, :] = -np.inf
    x[1, :] = np.nan
    x[2, 1:] = -np.inf
    x[3, ::2] = -np.inf
    x[4, ::3] = np.nan
    x[5, [7, 70, 700]] = np.inf
    x[6, :-1] = -np.inf
    x[7, :] = -3.4e38
    x[7, 11] = 3.4e38
    u = uniform(rows, 9)
    for par in (dict(), dict(temperature=0.0), dict(top_k=100), dict(top_p=0.7), dict(top_k=2, top_p=0.9, min_p=0.1)):
        got = run(dev(x), u, **par)
        check(x, u, got, *spelled(rows, par))
        assert got[0][0] == got[0][1] == -1 and got[1][0] == 0


def test_the_ends_of_the_random_numbers(frq):
    """u = 0 is the first that stays, the largest below 1 the last; numbers outside are held to that."""
    x = logits(1, 2000, 4).repeat(6, 1)
    u = np.array([0.0, 1 - 2.0 ** -24, 1.0, 7.0, -1.0, np.nan], np.float32)
    for par in (dict(), dict(top_k=9)):
        got = run(x.cuda(), u, **par)[0]
        t, k, p, m = (v[0] for v in spelled(1, par))
        stay = oracle(x[0].numpy(), 0.5, t, k, p, m)[2]
        assert got[0] == stay[0] == got[4] == got[5] and got[1] == got[2] == got[3] == stay[-1]


def test_parameters_out_of_range_in_arrays(frq):
    x, u = logits(6, 500, 5), uniform(6, 5)
    nan = float("nan")
    temp = np.array([-1, nan, np.inf, 1, 1, 1], np.float32)
    top_k = np.array([-3, 0, 0, -1, 0, 0], np.int32)
    top_p = np.array([1, 1, 1, 2, nan, -1], np.float32)
    min_p = np.array([0, 0, 0, -1, nan, 3], np.float32)
    got = run(x.cuda(), u, temperature=dev(temp), top_k=dev(top_k), top_p=dev(top_p), min_p=dev(min_p))
    check(x.numpy(), u, got, [0, 0, 1e30, 1, 1, 1], [0] * 6, [1, 1, 1, 1, 1, 0], [0, 0, 0, 0, 0, 1])


@pytest.mark.parametrize("dtype,ld", [("f32", 1003), ("bf16", 1001), ("f16", 1024)])
def test_strided_rows_on_a_stream(frq, dtype, ld):
    """A vocabulary's end that is padding is not read."""
    rows, vocab = 5, 1000
    x = logits(rows, ld, 6, dtype)
    x[:, vocab:] = 100.0
    u = uniform(rows, 6)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    xc = x.cuda()
    torch.cuda.synchronize()
    got = run(xc, u, dtype, ld=ld, vocab=vocab, stream=s, top_p=0.9)
    check(x.float().numpy()[:, :vocab], u, got, *spelled(rows, dict(top_p=0.9)))


def test_frequencies_follow_the_weights(frq):
    """4096 draws of one distribution over 8 tokens, the numbers a grid: every count is exact to one."""
    x = np.log(np.array([1, 2, 3, 4, 5, 6, 7, 8], np.float32))[None]
    n = 4096
    tok = run(dev(x.repeat(n, 0)), (np.arange(n, dtype=np.float32) + 0.5) / n)[0]
    p = np.arange(1, 9) / 36
    assert np.all(np.abs(np.bincount(tok, minlength=8) - n * p) <= 1.01)


def test_graph_replay_and_two_streams(frq):
    """Captured once, replayed on new logits and numbers; a second stream draws meanwhile."""
    rows, vocab = 3, 152064
    xs = [logits(rows, vocab, 10 + i) for i in range(4)]
    us = [uniform(rows, 10 + i) for i in range(4)]
    x, u = xs[0].cuda(), dev(us[0])
    tok, prob = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
    par = dict(top_k=50, top_p=0.95, temperature=0.75)
    s, other = device.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    device.sample(x, u, tok, rows, vocab, probs=prob, stream=s, **par)
    s.synchronize()
    with device.Graph.capture(s) as g:
        device.sample(x, u, tok, rows, vocab, probs=prob, stream=s, **par)
    for i in range(4):
        x.copy_(xs[i])
        u.copy_(torch.from_numpy(us[i]))
        y = xs[3 - i].cuda()
        torch.cuda.synchronize()
        g.launch(s)
        got = run(y, us[3 - i], stream=other, top_p=0.9)
        s.synchronize()
        check(xs[i].numpy(), us[i], (tok.cpu().numpy(), prob.cpu().numpy()), *spelled(rows, par))
        check(xs[3 - i].numpy(), us[3 - i], got, *spelled(rows, dict(top_p=0.9)))
    g.destroy()
    s.destroy()


def test_rows_past_32_bits(frq):
    vocab, ld = 5001, (1 << 30) + 4
    x = logits(3, vocab, 9, "bf16")
    wide = torch.zeros((3, ld), dtype=torch.bfloat16, device="cuda")
    wide[:, :vocab] = x.cuda()
    torch.cuda.synchronize()
    u = uniform(3, 9)
    for par in (dict(top_k=50, top_p=0.9), dict(temperature=0.0), dict(min_p=0.01)):
        check(x.float().numpy(), u, run(wide, u, "bf16", ld=ld, vocab=vocab, **par), *spelled(3, par))


def test_a_call_of_rows_and_the_rows_alone(frq):
    """Whole rows and slices of rows see the same weights and sums: the same tokens and probabilities."""
    rows, vocab = 140, 20011
    x, u = logits(rows, vocab, 10).cuda(), uniform(rows, 10)
    for par in (dict(), dict(top_k=300, top_p=0.95), dict(top_p=0.9, temperature=0.6, min_p=0.001), dict(top_k=3000)):
        tok, prob = run(x, u, **par)
        for i in (0, 77, 139):
            one = run(x[i:i + 1], u[i:i + 1], **par)
            assert one[0][0] == tok[i] and one[1][0] == prob[i], (i, par)
