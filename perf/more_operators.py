"""Timing cases of what a decoder runs between its projections, its cache and
its next token: what a caller of ``layer.DecoderProjections`` and
``attention.BlockAttention`` needs beside them.

Three operators:
  norm    add_rms_norm: the residual's addition and the root-mean-square norm
          behind it, out in 32 or 16 bits or as Q8_0 blocks
  chunk   attn_chunk: a chunk of new tokens of each sequence against the paged
          4-bit cache, which holds the chunk's own keys too
  sample  sample: one token per row of logits by temperature, top-k, top-p and
          min-p from a given random number

norm:   h = round(x + r) to the residual's type, y = h / sqrt(mean(h^2) + eps) w.
        Q8_0: y rounded to fp32; per 32 elements d = fp16(max|y| / 127), the
        quotient in fp32, code = round_even(y / d) held to +-127, value d code.
chunk:  query i of a sequence with n new tokens and length len sees the tokens
        j <= i + len - n; softmax(q k / sqrt(d)) v with the values the cache
        holds: 32 channels of a head of a token share d = fp16(-e / 8), e their
        element of largest magnitude (the first of equals), held to +-65504,
        code = min(15, max(0, round_even(x / d) + 8)), value d (code - 8).
sample: w = exp((x - max x) / T). Sorted by x (equal ones by index) the first
        top_k stay, of these the shortest run whose weights sum to top_p of
        theirs, of these the ones with w >= min_p. The token is the first, in
        the order of the indices, at which the sum of the weights that stayed
        exceeds u times all of it. T = 0: the largest, the lowest index of equals.
        Second output: the token's share of the weights that stayed.

``own`` False computes all of it in elementary torch operations, True calls
flatrun_amd.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "q8_0": 34 / 32}
BLOCK = 32                                   # elements that share a scale
EPS = 1e-6

# (query heads, key heads, head size) of the decoders this package is used with
HEADS = [(14, 2, 64), (16, 8, 128), (28, 4, 128), (32, 8, 128), (8, 4, 256)]
FREE = dict(temp=1.0, top_k=0, top_p=1.0, min_p=0.0)


def listed() -> list[dict]:
    return [
        # One token of a 0.5B model between two of its blocks: the smallest call.
        dict(name="norm_token", kind="norm", rows=1, hidden=896, src="f32", res="f32", out="f32"),
        # A prompt of an 8B model, handed to the bf16 GEMMs; residuals stay fp32.
        dict(name="norm_prompt", kind="norm", rows=8192, hidden=4096, src="f32", res="f32", out="bf16"),
        # An odd number of tokens of a 7B model, bf16 throughout, kept in 8 bits.
        dict(name="norm_q8", kind="norm", rows=4097, hidden=3584, src="bf16", res="bf16", out="q8_0"),
        # Five drafted tokens of a 0.5B model, checked after 1500: latency.
        dict(name="chunk_draft", kind="chunk", new="5", past="1500", hq=14, hkv=2, d=64, page=32, dtype="bf16", seed=1),
        # Thirty-two sequences, a few drafted tokens each, anywhere in their texts.
        dict(name="chunk_verify", kind="chunk", new="32x2-9", past="32x100-8000", hq=32, hkv=8, d=128, page=64,
             dtype="bf16", seed=2),
        # Prompts that come in pieces of up to 512 tokens, eight at a time.
        dict(name="chunk_prompts", kind="chunk", new="8x201-512", past="8x300-4096", hq=28, hkv=4, d=128, page=64,
             dtype="bf16", seed=3),
        # A short question about a long document: few rows, the whole cache.
        dict(name="chunk_document", kind="chunk", new="17", past="131000", hq=16, hkv=8, d=128, page=256, dtype="bf16",
             seed=4),
        # The next 2048 tokens of a long prompt: the largest product.
        dict(name="chunk_long", kind="chunk", new="2048", past="32768", hq=32, hkv=8, d=128, page=64, dtype="bf16",
             seed=5),
        # The next token of one sequence, the usual cuts: latency over a whole vocabulary.
        dict(name="sample_token", kind="sample", rows=1, vocab=152064, src="f32", each=False, temp=0.75, top_k=50,
             top_p=0.953125, min_p=0.0),
        # A few sequences of a model with a small vocabulary of odd size, bf16 logits with many equal ones.
        dict(name="sample_few", kind="sample", rows=7, vocab=32003, src="bf16", each=False, temp=1.25, top_k=0,
             top_p=1.0, min_p=0.0625),
        # A batch drawn from the whole distribution, as training on own samples does.
        dict(name="sample_whole", kind="sample", rows=64, vocab=131072, src="f32", each=False, **FREE),
        # A large batch, every request with parameters of its own, some of them greedy.
        dict(name="sample_mixed", kind="sample", rows=256, vocab=152064, src="f32", each=True, **FREE),
    ]


def _log(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    """One more case of the same ranges, no dearer than the largest listed one."""
    kind = rng.choice(["norm", "norm", "chunk", "chunk", "chunk", "sample", "sample"])
    if kind == "norm":
        hidden = _log(rng, 64, 16384)
        out = rng.choice(["f32", "bf16", "f16", "q8_0"])
        step = rng.choice([1, 8, 32]) if out != "q8_0" else BLOCK
        hidden = max(step, hidden // step * step)
        src = rng.choice(["f32", "f32", "bf16", "f16"])
        return dict(kind=kind, rows=_log(rng, 1, min(16384, 8192 * 4096 // hidden)), hidden=hidden, src=src,
                    res=rng.choice(["f32", src]), out=out)
    if kind == "sample":
        rows = _log(rng, 1, 256)
        vocab = _log(rng, 1000, 152064)
        each = rng.random() < 0.4
        par = FREE if each else dict(temp=rng.choice([0.0, 0.25, 0.75, 1.0, 1.5]), top_k=rng.choice([0, 0, 1, 40, 1000]),
                                     top_p=rng.choice([1.0, 0.984375, 0.90625, 0.5]),
                                     min_p=rng.choice([0.0, 0.0, 0.0625, 0.25]))
        return dict(kind=kind, rows=rows, vocab=vocab, src=rng.choice(["f32", "f32", "bf16", "f16"]), each=each, **par)
    hq, hkv, d = rng.choice(HEADS)
    n = _log(rng, 1, 32)
    hi = _log(rng, 1, 2048 // math.isqrt(n))
    lo = rng.choice([1, max(1, hi // 2), hi])
    # the scores of a batch stay below 2^31, the cache below 131072 tokens of eight heads of 128
    most = min(131072, (1 << 31) // (n * hi * hq) - hi, 131072 * 8 * 128 // (n * hkv * d))
    past = _log(rng, 1, max(1, most))
    low = rng.choice([0, past // 2, past])
    return dict(kind=kind, new=f"{n}x{lo}-{hi}", past=f"{n}x{low}-{past}", hq=hq, hkv=hkv, d=d,
                page=rng.choice([32, 64, 128, 256]), dtype="bf16", seed=rng.randrange(1 << 30))


def _lens(text: str, seed: int) -> list[int]:
    """"311" is one length, "16x2000-4096" sixteen of that range."""
    if "x" not in text:
        return [int(text)]
    n, span = text.split("x")
    lo, hi = map(int, span.split("-"))
    rng = random.Random(seed)
    return [rng.randint(lo, hi) for _ in range(int(n))]


def _chunk_lens(case) -> tuple[list[int], list[int]]:
    new, past = _lens(case["new"], case["seed"]), _lens(case["past"], case["seed"] + 1)
    return new, [a + b for a, b in zip(new, past)]


def work(case) -> dict:
    if case["kind"] == "norm":
        n = case["rows"] * case["hidden"]
        return {"bytes": int(n * (SIZE[case["src"]] + 2 * SIZE[case["res"]] + SIZE[case["out"]])) + 4 * case["hidden"],
                "flops": n * (5 if case["out"] != "q8_0" else 9)}
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * SIZE[case["src"]] + case["rows"] * 28, "flops": 4 * n}
    new, lens = _chunk_lens(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    held = 2 * hkv * (d // 2 + d // BLOCK * 2)
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, lens))
    return {"bytes": sum(lens) * held + 2 * sum(new) * hq * d * SIZE[case["dtype"]]
            + sum(4 * math.ceil(m / case["page"]) for m in lens) + 8 * len(lens), "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------ inputs

def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape) -> torch.Tensor:
    return torch.randn(shape, generator=g, device="cuda")


def _rand(g, *shape) -> torch.Tensor:
    return torch.rand(shape, generator=g, device="cuda")


def _pick(g, rows: int, values: list) -> torch.Tensor:
    """One of the values for each row."""
    return torch.tensor(values, device="cuda")[torch.randint(0, len(values), (rows,), generator=g, device="cuda")]


def _norm_inputs(case, g) -> dict:
    n, hidden = case["rows"], case["hidden"]
    # residuals have a size per channel, a few channels far above the others
    ch = torch.exp(0.5 * _randn(g, hidden))
    ch = torch.where(_rand(g, hidden) < 0.004, 30 * ch, ch)
    return {"x": (_randn(g, n, hidden) * 0.4).to(DT[case["src"]]), "r": (_randn(g, n, hidden) * ch).to(DT[case["res"]]),
            "w": 1 + 0.3 * _randn(g, hidden)}


def _sample_inputs(case, g) -> dict:
    n, vocab = case["rows"], case["vocab"]
    # most of a vocabulary far below the few tokens that fit, in some rows more of them
    x = 2 * _randn(g, n, vocab) + (1 + 2 * _rand(g, n, 1)) * torch.where(_rand(g, n, vocab) < 20 / vocab, 5.0, 0.0)
    x = torch.where(_rand(g, vocab) < 0.002, float("-inf"), x)                    # ids that stand for nothing
    if case["each"]:
        par = {"temp": _pick(g, n, [0.0, 0.3, 0.7, 1.0, 1.3]), "top_k": _pick(g, n, [0, 0, 1, 40, 1000]).int(),
               "top_p": _pick(g, n, [1.0, 0.98, 0.9, 0.5]), "min_p": _pick(g, n, [0.0, 0.0, 0.02, 0.1])}
    else:
        par = {p: case[p] for p in FREE}
    return {"x": x.to(DT[case["src"]]), "u": _rand(g, n), "par": par}


def _chunk_inputs(case, g) -> dict:
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    new, lens = _chunk_lens(case)
    # pages in shuffled order: the table of each sequence, and the slot of every token
    per = [max(1, math.ceil(m / page)) for m in lens]
    perm = torch.randperm(sum(per), generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(lens), max(per)), dtype=torch.int32, device="cuda")
    slots, at = [], 0
    for i, (m, p) in enumerate(zip(lens, per)):
        table[i, :p] = perm[at:at + p]
        t = torch.arange(m, device="cuda")
        slots.append(table[i, t // page].long() * page + t % page)
        at += p
    # a size per channel of each head, a few of them large, as keys have them
    ch = torch.exp(0.4 * _randn(g, hkv, d))
    ch = torch.where(_rand(g, hkv, d) < 1 / 64, 6 * ch, ch)
    k = _randn(g, sum(lens), hkv, d) * ch
    v = _randn(g, sum(lens), hkv, d) * (0.5 + _rand(g, hkv, d))
    q = (1.5 * _randn(g, sum(new), hq, d) / ch.repeat_interleave(hq // hkv, 0)).to(DT[case["dtype"]])
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
    return {"k": k, "v": v, "q": q, "new": new, "lens": lens, "table": table, "slots": torch.cat(slots),
            "pages": sum(per), "cu_q": cu, "lens_dev": torch.tensor(lens, dtype=torch.int32, device="cuda")}


def _inputs(case, seed) -> dict:
    """The inputs, from the seed alone."""
    make = {"norm": _norm_inputs, "chunk": _chunk_inputs, "sample": _sample_inputs}[case["kind"]]
    return make(case, _gen(seed))


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    kind = case["kind"]
    if own:
        if kind == "norm":
            n, hidden = case["rows"], case["hidden"]
            st["sum"] = torch.empty_like(st["r"])
            st["out"] = (torch.empty((n, hidden // BLOCK, 34), dtype=torch.uint8, device="cuda") if case["out"] == "q8_0"
                         else torch.empty((n, hidden), dtype=DT[case["out"]], device="cuda"))
            st["val"] = torch.empty((n, hidden), device="cuda") if case["out"] == "q8_0" else None
        elif kind == "sample":
            st["tok"] = torch.empty(case["rows"], dtype=torch.int32, device="cuda")
            st["prob"] = torch.empty(case["rows"], device="cuda")
        else:
            from flatrun_amd.attention import KVCache4

            # what earlier steps, and the projection of this one, left in the cache
            st["cache"] = c = KVCache4(st["pages"], case["page"], case["hkv"], case["d"])
            c.write(st.pop("k"), st.pop("v"), st["slots"], st["slots"].numel(), dtype="f32",
                    stream=torch.cuda.current_stream())
            st["out"] = torch.empty_like(st["q"])
        torch.cuda.synchronize()             # the inputs are there, whatever stream reads them
    elif kind == "chunk":
        n = st["pages"] * case["page"]
        for p in "kv":
            x = st.pop(p)
            st[p + "c"] = torch.zeros((n, case["hkv"], case["d"] // 2), dtype=torch.uint8, device="cuda")
            st[p + "d"] = torch.zeros((n, case["hkv"], case["d"] // BLOCK), dtype=torch.float16, device="cuda")
            b = x.view(x.shape[0], x.shape[1], -1, BLOCK)
            d = (b.gather(-1, b.abs().argmax(-1, keepdim=True)) / -8).clamp(-65504, 65504).half()
            f = d.float()
            code = torch.where(f == 0, 8.0, (torch.round(b / f) + 8).clamp(0, 15)).to(torch.uint8)
            st[p + "c"][st["slots"]] = (code[..., 0::2] | (code[..., 1::2] << 4)).view(x.shape[0], x.shape[1], -1)
            st[p + "d"][st["slots"]] = d[..., 0]
        # where each place of the batch's longest sequence is: behind a shorter one's end, its first token
        t = torch.arange(max(st["lens"]), device="cuda")
        t = torch.where(t < st["lens_dev"][:, None], t, 0)
        st["at"] = st["table"].long().gather(1, t // case["page"]) * case["page"] + t % case["page"]
        # which query of which sequence stands in each row of a padded batch
        i = torch.arange(max(st["new"]), device="cuda")
        counts = (st["cu_q"][1:] - st["cu_q"][:-1])[:, None]
        st["real"] = i < counts
        st["row"] = torch.where(st["real"], st["cu_q"][:-1, None] + i, 0).long()
    return st


# -------------------------------------------------------------- plain forms

def _norm_plain(st) -> list:
    case = st["case"]
    h = (st["x"].float() + st["r"].float()).to(DT[case["res"]])
    if case["out"] != "q8_0":
        f = h.float()
        y = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * st["w"]
        return [h, y.to(DT[case["out"]])]
    f = h.double()                           # a code is next to a border now and then
    y = (f / torch.sqrt((f * f).mean(-1, keepdim=True) + EPS) * st["w"].double()).float()
    b = y.view(y.shape[0], -1, BLOCK)
    d = (b.abs().amax(-1, keepdim=True) / 127).half().float()
    code = torch.where(d == 0, 0.0, torch.round(b.double() / d.double()).clamp(-127, 127).float())
    return [h, (code * d).view(y.shape)]


def _values(st, p: str) -> torch.Tensor:
    """What the cache holds for every place of the padded batch."""
    c, d = st[p + "c"][st["at"]], st[p + "d"][st["at"]]
    code = torch.stack([c & 15, c >> 4], dim=-1).float().view(*d.shape, BLOCK) - 8
    return (code * d.float()[..., None]).flatten(-2)                              # sequence, token, head, channel


def _chunk_plain(st) -> torch.Tensor:
    case = st["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    q = st["q"].float()[st["row"]]                                                # sequence, query, head, channel
    b, m = q.shape[:2]
    q = q.view(b, m, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    k = _values(st, "k").permute(0, 2, 3, 1).contiguous()
    s = torch.matmul(q, k).view(b, hkv, -1, m, k.shape[-1])
    del k
    last = (st["lens_dev"] - (st["cu_q"][1:] - st["cu_q"][:-1]))[:, None] + torch.arange(m, device="cuda")
    unseen = torch.arange(s.shape[-1], device="cuda") > last[..., None]
    s.mul_(1 / math.sqrt(d)).masked_fill_(unseen[:, None, None], float("-inf"))
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    s.div_(s.sum(-1, keepdim=True))
    v = _values(st, "v").transpose(1, 2).contiguous()
    o = torch.matmul(s.view(b, hkv, -1, s.shape[-1]), v).view(b, hkv, -1, m, d)
    return o.permute(0, 3, 1, 2, 4).reshape(b, m, hq, d)[st["real"]].to(DT[case["dtype"]])


def _sample_plain(st) -> list:
    # in 64 bits: a sum's last bits decide between neighbouring tokens
    x = st["x"].double()
    rows, vocab = x.shape
    par = {p: torch.as_tensor(v, device="cuda").double().reshape(-1, 1) for p, v in st["par"].items()}
    x, index = torch.sort(x, dim=-1, descending=True, stable=True)
    greedy = (par["temp"] == 0).expand(rows, 1)
    w = torch.exp((x - x[:, :1]) / torch.where(par["temp"] == 0, 1.0, par["temp"]))
    place = torch.arange(vocab, device="cuda")
    w = torch.where(greedy, (place == 0).double(), w)
    w = torch.where((par["top_k"] > 0) & (place >= par["top_k"]), 0.0, w)
    upto = torch.cumsum(w, -1)
    before = torch.cat([torch.zeros_like(upto[:, :1]), upto[:, :-1]], dim=-1)
    stay = (before < par["top_p"] * upto[:, -1:]) | (par["top_p"] >= 1) | (place == 0)
    w = torch.where(stay & (w >= par["min_p"]), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, index, w)
    upto = torch.cumsum(w, -1)
    token = (upto <= st["u"].double()[:, None] * upto[:, -1:]).sum(-1)
    token = torch.minimum(token, torch.where(w > 0, place, 0).amax(-1))
    return [token.int(), (w.gather(1, token[:, None]) / upto[:, -1:])[:, 0].float()]


# -------------------------------------------------------------------- passes

def run(st):
    case = st["case"]
    kind = case["kind"]
    if not own:
        return {"norm": _norm_plain, "chunk": _chunk_plain, "sample": _sample_plain}[kind](st)
    from flatrun_amd import device

    s = torch.cuda.current_stream()
    if kind == "norm":
        device.add_rms_norm(st["x"], st["out"], case["rows"], case["hidden"], weight=st["w"], residual=st["r"],
                            sum_out=st["sum"], eps=EPS, x_dtype=case["src"], res_dtype=case["res"],
                            out_dtype=case["out"], stream=s)
        if case["out"] != "q8_0":
            return [st["sum"], st["out"]]
        device.dequant("Q8_0", st["out"], st["val"], case["rows"] * case["hidden"], stream=s)
        return [st["sum"], st["val"]]
    if kind == "sample":
        p = st["par"]
        device.sample(st["x"], st["u"], st["tok"], case["rows"], case["vocab"], temperature=p["temp"], top_k=p["top_k"],
                      top_p=p["top_p"], min_p=p["min_p"], probs=st["prob"], dtype=case["src"], stream=s)
        return [st["tok"], st["prob"]]
    device.attn_chunk(st["q"], st["cache"], st["table"], st["lens_dev"], st["cu_q"], st["out"], len(st["new"]),
                      sum(st["new"]), case["hq"], max_q=max(st["new"]), max_len=max(st["lens"]), dtype=case["dtype"],
                      stream=s)
    return st["out"]


# --------------------------------------------------------------- definitions

def _block_values(x: torch.Tensor) -> torch.Tensor:
    """What the 4-bit block keeps of x, block by block: the definition. The
    scale is an fp16 number by definition; everything else is in 64 bits."""
    b = x.double().reshape(-1, BLOCK)
    top = b.abs().amax(dim=1, keepdim=True)
    first = (b.abs() == top).to(torch.int8).argmax(dim=1)
    e = b[torch.arange(b.shape[0], device=b.device), first]
    d = torch.clamp(-e / 8, -65504, 65504).to(torch.float16).double()[:, None]
    level = torch.clamp(torch.round(b / torch.where(d == 0, 1.0, d)), -8, 7)
    return (torch.where(d == 0, 0.0, level) * d).reshape(x.shape)


def _draw_exactly(x: np.ndarray, u: float, temp: float, top_k: int, top_p: float, min_p: float) -> float:
    """The drawn token's share, one row at a time."""
    if temp == 0:
        return 1.0
    w = np.exp((x - x.max()) / temp)
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[:top_k] if top_k > 0 else order
    if top_p < 1:
        upto = np.cumsum(w[order])
        order = order[:1 + int(np.searchsorted(upto, top_p * upto[-1], side="left"))]
    order = np.sort(order[w[order] >= min_p])
    upto = np.cumsum(w[order])
    at = min(int(np.searchsorted(upto, u * upto[-1], side="right")), int(np.flatnonzero(w[order]).max()))
    return w[order[at]] / upto[-1]


def exact(case, seed):
    st = _inputs(case, seed)
    if case["kind"] == "norm":
        h = (st["x"].double() + st["r"].double()).to(DT[case["res"]]).double()
        y = st["w"].double() * h / torch.sqrt(h.square().sum(-1, keepdim=True) / case["hidden"] + EPS)
        if case["out"] == "q8_0":            # in fp32 by definition, and its scale in fp16
            b = y.to(torch.float32).reshape(-1, BLOCK)
            d = (b.abs().max(dim=1, keepdim=True).values / 127).to(torch.float16).double()
            level = torch.round(b.double() / torch.where(d == 0, 1.0, d)).clamp(-127, 127)
            y = (level * d).reshape(y.shape)
        return [h, y]
    if case["kind"] == "sample":
        x, u = st["x"].double().cpu().numpy(), st["u"].double().cpu().numpy()
        n = case["rows"]
        par = [np.broadcast_to(np.asarray(v.cpu() if torch.is_tensor(v) else v), (n,)) for v in st["par"].values()]
        share = [_draw_exactly(x[i], u[i], float(par[0][i]), int(par[1][i]), float(par[2][i]), float(par[3][i]))
                 for i in range(n)]
        return [None, np.array(share)]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    k, v = (torch.cat([_block_values(x) for x in st[p].split(1 << 15)]) for p in "kv")
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    aq = ak = 0
    for n, m in zip(st["new"], st["lens"]):
        for h in range(hq):
            kh, vh = k[ak:ak + m, h * hkv // hq], v[ak:ak + m, h * hkv // hq]
            s = st["q"][aq:aq + n, h].double() @ kh.t().contiguous() / math.sqrt(d)
            s = s + torch.full((n, m), float("-inf"), dtype=torch.float64, device="cuda").triu(m - n + 1)
            out[aq:aq + n, h] = torch.exp(s - torch.logsumexp(s, -1, keepdim=True)) @ vh
        aq, ak = aq + n, ak + m
    return out
