"""A small decoder's steps with every operator on the device, from the embedding
rows to the tokens: norm, projections, attention on the cache (prompts, chunks
straight from the cache, single tokens), residual and norm, MLP, vocabulary,
draw. Each stage is held against its 64-bit form on the stage's own input, as
its own tests do: projections within 1e-5, the norm half a last place and 2^-30,
the attention's bound beside its check, tokens equal."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from attn_ref import TORCH, attend, f64, fp32_bound, rope
from conftest import assert_matvec_close
from flatrun_amd import device, synth
from flatrun_amd.attention import BlockAttention, KVCache4, Sequence, rope_table
from flatrun_amd.layer import DecoderProjections, Residual
from flatrun_amd.sampling import Sampler
from oracle import gguf_np as G
from test_gpu_attention_layers import bf16, cached, upload
from test_gpu_norm import oracle as norm
from test_gpu_sample import oracle as draw

pytestmark = pytest.mark.gpu

HQ, HKV, D, HIDDEN, INTER, VOCAB, LAYERS = 4, 2, 64, 256, 512, 1000, 2
SHAPES = {"q": ("Q4_K", HQ * D, HIDDEN), "k": ("Q4_K", HKV * D, HIDDEN), "v": ("Q6_K", HKV * D, HIDDEN),
          "o": ("Q4_K", HIDDEN, HQ * D), "gate": ("Q4_K", INTER, HIDDEN), "up": ("Q4_K", INTER, HIDDEN),
          "down": ("Q6_K", HIDDEN, INTER)}


class Decoder:
    def __init__(self, direct=True, max_rows=96, seed=3):
        rng = np.random.default_rng(seed)
        up = device.DeviceBuffer.from_host
        self.direct, self.stream, self.positions = direct, device.Stream(), rope_table(D, 512)
        self.host = [{n: synth.make_blocks(q, m, k, seed=seed + 10 * i + j) for j, (n, (q, m, k)) in enumerate(SHAPES.items())}
                     for i in range(LAYERS)]
        self.head = synth.make_blocks("Q6_K", VOCAB, HIDDEN, seed=seed + 99)
        self.norms = [(1 + 0.2 * rng.standard_normal(HIDDEN)).astype(np.float32) for _ in range(2 * LAYERS + 1)]
        self.dev_norms = [up(w) for w in self.norms]
        self.caches = [KVCache4(24, 32, HKV, D) for _ in range(LAYERS)]
        self.blocks, self.steps = [], []
        table = up(self.positions)
        for host, cache in zip(self.host, self.caches):
            dev = {n: up(raw) for n, raw in host.items()}
            self.blocks.append(DecoderProjections({n: (q, dev[n], m, k, host[n].nbytes) for n, (q, m, k) in SHAPES.items()},
                                                  max_seq=max_rows, stream=self.stream))
            kw = {"first": self.steps[0]} if self.steps else dict(max_rows=max_rows, max_seqs=3, max_context=300,
                                                                  stream=self.stream, direct=direct)
            self.steps.append(BlockAttention(cache, HQ, table, 512, **kw))
        self.dev_head = up(self.head)
        self.residual = Residual(HIDDEN, max_rows, stream=self.stream)
        self.sampler = Sampler(VOCAB, 3, stream=self.stream)
        self.x, self.logits = device.DeviceBuffer(4 * HIDDEN * max_rows), device.DeviceBuffer(4 * VOCAB * 3)
        self.last, self.u = device.DeviceBuffer(4 * HIDDEN * 3), device.DeviceBuffer(4 * 3)

    def forward(self, rows, ends, see=lambda what, buf, *a: None):
        """ends: each sequence's last row."""
        r = self.residual
        xn = r.start(self.x, self.dev_norms[0], rows)
        see("norm", xn, self.x, 0)
        for i, (block, step) in enumerate(zip(self.blocks, self.steps)):
            def attention(qkv, n):
                see("qkv", qkv, xn, i)
                out = step(qkv, n)
                see("attention", out, qkv, i)
                return out

            def after(o, n):
                see("o", o, step.out, i)
                see("residual", r.rows)
                got = r.add(o, self.dev_norms[2 * i + 1], n)
                see("add", got, o, 2 * i + 1)
                return got

            out = block.forward(xn, rows, attention=attention, post_attention=after)
            see("mlp", out, xn, i)
            see("residual", r.rows)
            xn = r.add(out, self.dev_norms[2 * i + 2], rows)
            see("add", xn, out, 2 * i + 2)
        for i, e in enumerate(ends):
            device.copy(self.last.ptr + 4 * HIDDEN * i, xn.ptr + 4 * HIDDEN * e, 4 * HIDDEN, stream=self.stream)
        device.gemv("Q6_K", self.dev_head, self.last, self.logits, VOCAB, HIDDEN, batch=len(ends), stream=self.stream,
                    w_bytes=self.head.nbytes)
        return self.sampler(self.logits, self.u, len(ends))

    def close(self):
        for b in (*self.blocks, self.steps[0], *self.caches, self.residual, self.sampler):
            b.close()


class Look:
    """Checks each stage on its own input."""

    def __init__(self, net, new, start):
        self.net, self.new, self.start, self.rows = net, new, start, sum(new.values())

    def fetch(self, buf, width):
        self.net.stream.synchronize()
        return buf.to_host(np.float32)[:self.rows * width].reshape(self.rows, width)

    def close_to(self, name, i, x, y):
        q, n, k = SHAPES[name]
        raw = self.net.host[i][name]
        y64, size = G.matmul_f64(q, x, raw, n, k), G.abs_matmul_f64(q, x, raw, n, k)
        for a, b, c in zip(y, y64, size):
            assert_matvec_close(a, b, c, what=f"{name} of block {i}")

    def __call__(self, what, buf, src=None, i=None):
        net = self.net
        if what == "residual":
            self.before = self.fetch(buf, HIDDEN)
        elif what in ("norm", "add"):
            h = self.fetch(src, HIDDEN)
            if what == "add":
                h = h + self.before
                assert np.array_equal(h, self.fetch(net.residual.rows, HIDDEN))
            want = norm(torch.as_tensor(h), net.norms[i], 1e-6)
            assert np.all(np.abs(self.fetch(buf, HIDDEN) - want) <= (2.0 ** -24 + 2.0 ** -30) * np.abs(want) + 1e-44), (what, i)
        elif what == "qkv":
            x, y = self.fetch(src, HIDDEN), self.fetch(buf, (HQ + 2 * HKV) * D)
            for name, a, b in zip("qkv", (0, HQ * D, (HQ + HKV) * D), (HQ * D, (HQ + HKV) * D, (HQ + 2 * HKV) * D)):
                self.close_to(name, i, x, y[:, a:b])
        elif what == "o":
            self.close_to("o", i, self.fetch(src, HQ * D), self.fetch(buf, HIDDEN))
        elif what == "mlp":
            gateup = self.fetch(net.blocks[i].gateup, 2 * INTER) if self.rows > 1 else None
            x, act = self.fetch(net.residual.xn, HIDDEN), self.fetch(net.blocks[i].act, INTER)
            if gateup is not None:
                self.close_to("gate", i, x, gateup[:, :INTER])
                self.close_to("up", i, x, gateup[:, INTER:])
            self.close_to("down", i, act, self.fetch(buf, HIDDEN))
        else:
            self.attention(self.fetch(src, (HQ + 2 * HKV) * D), self.fetch(buf, HQ * D).reshape(-1, HQ, D), i)

    def heads(self, i, dtype, count):
        """q, k and v of the step's rows once more: the same launch, so the same bits."""
        step, p = self.net.steps[i], self.net.steps[0]._plan
        q, k, v = (torch.empty((count, h, D), dtype=TORCH[dtype], device="cuda") for h in (HQ, HKV, HKV))
        device.qk_norm_rope(self.net.blocks[i].qkv, q, k, v, count, HQ, HKV, D, step.table, p["positions"], out_dtype=dtype, n_pos=512)
        torch.cuda.synchronize()
        return f64(q), f64(k), f64(v)

    def attention(self, qkv, got, i):
        """The synthetic weights make scores of hundreds, so q and k are taken as the products have them
        (rounded to bf16 or fp16 from the same values) and only the sums' error is left to a score: fp32_bound's,
        with the exponential in place of its first term, exp(2 e) - 1. A weight is rounded for its product, its
        sum may be of the rounded ones: twice half a last place, and for fp16 2^-30 of the largest. attn_decode keeps
        a weight times a scale (an eighth of a block's largest value, under codes up to 8) to 2^-40 of the largest
        of either: 2^-40 of the largest value for each token."""
        net, at = self.net, 0
        context = any(self.start[s] and n > 1 for s, n in self.new.items())
        made = {t: self.heads(i, t, self.rows) for t in ("f32", "bf16")}
        for s, n in self.new.items():
            pos = np.arange(self.start[s], s.length)
            want, size = rope(qkv[at:at + n].reshape(n, -1, D), HQ, HKV, D, D, False, net.positions[pos])
            kind = "f32" if n == 1 else "bf16"
            q, k, v = (x[at:at + n] for x in made[kind])
            for x, w, m in zip((q, k, v), want, size):
                assert np.all(np.abs(x - w) <= 20 * 2.0 ** -24 * m + (n > 1) * 2.0 ** -8 * 1.001 * np.abs(w) + 2.0 ** -25)
            ck, cv = cached(net.caches[i], s)
            weight = 2.0 ** -8
            if n == 1:
                kk, vv, weight = ck, cv, 0
            elif not context:
                kk, vv = k, v
            elif net.direct:
                kk, vv, weight = half(ck), half(cv), 2.0 ** -11
            else:
                kk, vv = bf16(ck), bf16(cv)
            for h in range(HQ):
                g = h // (HQ // HKV)
                want, mag, size = attend(q[:, h], kk[:, g], vv[:, g], D ** -0.5, pos)
                score = fp32_bound(np.ones(1), size, 0, D) / 2
                tol = (np.expm1(2 * score) + fp32_bound(np.ones(1), 0 * size, len(kk), D) + 2 * weight) * mag
                tol = tol + {2.0 ** -11: 2.0 ** -29, 0: 2.0 ** -40}.get(weight, 0) * len(kk) * np.abs(vv).max()
                err = np.abs(got[at:at + n, h] - want)
                assert np.all(err <= tol + 1e-30), (n, self.start[s], h, float((err / np.maximum(tol, 1e-30)).max()))
            at += n


def half(a):
    return a.astype(np.float16).astype(np.float64)


PARAMS = [dict(temperature=0.8, top_k=40, top_p=0.95), dict(temperature=0.0), dict(top_p=0.9, min_p=0.02)]


@pytest.mark.parametrize("direct", [True, False])
def test_every_stage(frq, direct):
    rng = np.random.default_rng(5)
    net = Decoder(direct)
    a, b, c = (Sequence() for _ in range(3))
    for new in ({a: 45, b: 7}, {a: 40, b: 1, c: 5}, {a: 1, b: 1, c: 1}, {b: 30, c: 66}, {a: 1, c: 3}, {a: 1}):
        rows, start = sum(new.values()), {s: s.length for s in new}
        upload(net.x, rng.standard_normal((rows, HIDDEN)).astype(np.float32))
        u = rng.random(3, dtype=np.float32)
        upload(net.u, u)
        net.steps[0].plan(new)
        net.sampler.plan(PARAMS[:len(new)])
        ends = (np.cumsum(list(new.values())) - 1).tolist()
        tokens = net.forward(rows, ends, Look(net, new, start))
        net.stream.synchronize()
        last = net.residual.xn.to_host(np.float32).reshape(-1, HIDDEN)[ends]
        logits = net.logits.to_host(np.float32).reshape(-1, VOCAB)[:len(ends)]
        for y, y64, size in zip(logits, G.matmul_f64("Q6_K", last, net.head, VOCAB, HIDDEN),
                                G.abs_matmul_f64("Q6_K", last, net.head, VOCAB, HIDDEN)):
            assert_matvec_close(y, y64, size, what="vocabulary")
        for i, (tok, p) in enumerate(zip(tokens.to_host(np.int32), net.sampler.probs.to_host(np.float32)[:len(ends)])):
            par = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) | PARAMS[i]
            want, share, _ = draw(logits[i], float(u[i]), *(x if k == "top_k" else float(np.float32(x)) for k, x in par.items()))
            assert tok == want and abs(p - share) <= 2.0 ** -23 * share + 1e-9, (i, new)
    net.close()


def test_a_captured_step(frq):
    """Single tokens, the whole step captured once: after each later plan the replay has the eager step's bits."""
    rng = np.random.default_rng(6)
    net = Decoder()
    seqs = [Sequence(), Sequence()]
    upload(net.x, rng.standard_normal((67, HIDDEN)).astype(np.float32))
    upload(net.u, rng.random(3, dtype=np.float32))
    net.steps[0].plan({seqs[0]: 60, seqs[1]: 7})
    net.sampler.plan(PARAMS[:2])
    net.forward(67, [59, 66])
    net.stream.synchronize()
    graph, seen = None, set()
    for i in range(40):
        x = rng.standard_normal((2, HIDDEN)).astype(np.float32)
        upload(net.u, rng.random(3, dtype=np.float32))
        net.steps[0].plan({s: 1 for s in seqs}, max_len=300)
        net.sampler.plan([PARAMS[i % 3], PARAMS[(i + 1) % 3]])
        upload(net.x, x)
        if graph is None:
            net.forward(2, [0, 1])
            net.stream.synchronize()
            with device.Graph.capture(net.stream) as graph:
                net.forward(2, [0, 1])
        got = []
        for run in (lambda: graph.launch(net.stream), lambda: net.forward(2, [0, 1])):
            upload(net.x, x)
            run()
            net.stream.synchronize()
            got.append((net.sampler.tokens.to_host(np.int32)[:2], net.logits.to_host(np.float32)[:2 * VOCAB]))
        assert np.isfinite(got[0][1]).all() and np.array_equal(got[0][1], got[1][1]), i
        assert np.array_equal(got[0][0], got[1][0]), i
        seen.update(got[0][0].tolist())
    assert len(seen) > 5
    graph.destroy()
    net.close()
