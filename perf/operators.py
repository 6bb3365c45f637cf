"""Timing cases of the attention step of a decoder block: what runs between
the q|k|v projection and the o projection of ``layer.DecoderProjections``.

Four operators:
  rope     qk_norm_rope: the norm of every query and key head and the rotary
           position in one pass over the q|k|v rows of the projection
  kv       KVCache4.write and .read: keys and values quantised to 4 bits as
           they enter a paged cache, and the values they stand for read back
  decode   attn_decode: one query token per sequence against the paged cache
  prefill  attn_prefill: causal attention over packed sequences of different
           lengths, keys possibly longer than queries (a prompt in chunks)

The 4-bit block: 32 channels of one head of one token; e its element of the
largest magnitude (the first of equals), d = fp16(-e / 8) held to +-65504,
code = min(15, max(0, round_to_even(x / d) + 8)), the value d * (code - 8).

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
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 32                                   # channels that share a scale
TABLE = 32768                                # positions in the rotary table
EPS = 1e-6

# (query heads, key heads, head size) of the decoders this package is used with
HEADS = [(14, 2, 64), (16, 8, 128), (28, 4, 128), (32, 8, 128), (8, 4, 256)]


def listed() -> list[dict]:
    return [
        # One token of a 0.5B model: the smallest call, launch and latency.
        dict(name="rope_token", kind="rope", tokens=1, hq=14, hkv=2, d=64, rot=64, pairs="half", norm=False,
             src="f32", out="f32", seed=1),
        # A prompt of an 8B model with normed heads, handed to the prompt's attention in bf16.
        dict(name="rope_prompt", kind="rope", tokens=8192, hq=32, hkv=8, d=128, rot=128, pairs="half", norm=True,
             src="f32", out="bf16", seed=2),
        # Interleaved pairs over a quarter of a large head, an odd number of tokens, bf16 in and out.
        dict(name="rope_partial", kind="rope", tokens=1001, hq=8, hkv=4, d=256, rot=64, pairs="interleaved",
             norm=False, src="bf16", out="bf16", seed=3),
        # Sixty-four sequences each add the token they just computed.
        dict(name="kv_append", kind="kv", tokens=64, hkv=8, d=128, page=64, src="f32", out="f32", seed=4),
        # A prompt enters the cache; a later chunk reads it back.
        dict(name="kv_prompt", kind="kv", tokens=8192, hkv=8, d=128, page=64, src="bf16", out="bf16", seed=5),
        # One sequence of a 0.5B model, a few hundred tokens in: latency again.
        dict(name="decode_short", kind="decode", lens="311", hq=14, hkv=2, d=64, page=32, dtype="f32", seed=6),
        # A 7B model, sixteen sequences of similar length, bf16 activations.
        dict(name="decode_batch", kind="decode", lens="16x2000-4096", hq=28, hkv=4, d=128, page=64, dtype="bf16",
             seed=7),
        # An 8B model serving sixty-four sequences anywhere between their first token and 8K.
        dict(name="decode_ragged", kind="decode", lens="64x1-8192", hq=32, hkv=8, d=128, page=64, dtype="f32",
             seed=8),
        # One long document: a single sequence must fill the whole GPU.
        dict(name="decode_long", kind="decode", lens="131072", hq=32, hkv=8, d=128, page=256, dtype="f32", seed=9),
        # A short prompt of a 7B model, an odd number of tokens.
        dict(name="prefill_short", kind="prefill", lens="333", past="0", hq=28, hkv=4, d=128, dtype="bf16",
             causal=True, seed=10),
        # Prompts of different lengths packed together, some of them the next chunk of a longer one.
        dict(name="prefill_packed", kind="prefill", lens="24x17-1500", past="24x0-1200", hq=32, hkv=8, d=128,
             dtype="bf16", causal=True, seed=11),
        # A long prompt of an 8B model: the largest product.
        dict(name="prefill_long", kind="prefill", lens="16384", past="0", hq=32, hkv=8, d=128, dtype="bf16",
             causal=True, seed=12),
    ]


def _log(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    """One more case of the same ranges, no dearer than the largest listed one."""
    kind = rng.choice(["rope", "kv", "decode", "decode", "prefill", "prefill"])
    hq, hkv, d = rng.choice(HEADS)
    seed = rng.randrange(1 << 30)
    if kind == "rope":
        tokens = _log(rng, 1, 8192)
        return dict(kind=kind, tokens=tokens, hq=hq, hkv=hkv, d=d, rot=d // rng.choice([1, 1, 2, 4]),
                    pairs=rng.choice(["half", "interleaved"]), norm=rng.random() < 0.5,
                    src=rng.choice(["f32", "f32", "bf16"]), out=rng.choice(["f32", "bf16", "f16"]), seed=seed)
    if kind == "kv":
        src = rng.choice(["f32", "bf16", "f16"])
        return dict(kind=kind, tokens=_log(rng, 1, 8192), hkv=hkv, d=d, page=rng.choice([32, 64, 128, 256]), src=src,
                    out=rng.choice(["f32", src]), seed=seed)
    if kind == "decode":
        batch = _log(rng, 1, 64)
        most = min(131072, (1 << 18) * 8 * 128 // (batch * hkv * d))
        hi = _log(rng, 1, most)
        lo = rng.choice([0, 1, hi // 2, hi])
        return dict(kind=kind, lens=f"{batch}x{min(lo, hi)}-{hi}", hq=hq, hkv=hkv, d=d,
                    page=rng.choice([32, 64, 128, 256]), dtype=rng.choice(["f32", "f32", "bf16", "f16"]), seed=seed)
    n = _log(rng, 1, 32)
    hi = _log(rng, 1, 8192 // math.isqrt(n))
    lo = rng.choice([1, max(1, hi // 2), hi])
    past = rng.choice([0, 0, _log(rng, 1, 1024)])
    return dict(kind=kind, lens=f"{n}x{lo}-{hi}", past=f"{n}x0-{past}", hq=hq, hkv=hkv, d=d,
                dtype=rng.choice(["bf16", "bf16", "f16"]), causal=rng.random() < 0.8, seed=seed)


def _lens(text: str, seed: int) -> list[int]:
    """"311" is one length, "16x2000-4096" sixteen of that range."""
    if "x" not in text:
        return [int(text)]
    n, span = text.split("x")
    lo, hi = map(int, span.split("-"))
    rng = random.Random(seed)
    return [rng.randint(lo, hi) for _ in range(int(n))]


def _pairs(case) -> int:
    """Query-key pairs that a prompt's mask leaves."""
    total = 0
    for nq, past in zip(_lens(case["lens"], case["seed"]), _lens(case["past"], case["seed"] + 1)):
        total += nq * past + nq * (nq + 1) // 2 if case["causal"] else nq * (nq + past)
    return total


def work(case) -> dict:
    kind, hkv, d = case["kind"], case["hkv"], case["d"]
    if kind == "rope":
        n = case["tokens"] * (case["hq"] + 2 * hkv) * d
        rows = min(case["tokens"], TABLE)
        return {"bytes": n * (SIZE[case["src"]] + SIZE[case["out"]]) + rows * case["rot"] * 4 + case["tokens"] * 4,
                "flops": n * (7 if case["norm"] else 3)}
    if kind == "kv":
        n = 2 * case["tokens"] * hkv * d
        held = n // 2 + n // BLOCK * 2
        return {"bytes": n * (SIZE[case["src"]] + SIZE[case["out"]]) + 2 * held + 8 * case["tokens"], "flops": 6 * n}
    if kind == "decode":
        lens = _lens(case["lens"], case["seed"])
        held = 2 * hkv * (d // 2 + d // BLOCK * 2)
        return {"bytes": sum(lens) * held + len(lens) * 2 * case["hq"] * d * SIZE[case["dtype"]]
                + sum(4 * math.ceil(n / case["page"]) for n in lens) + 4 * len(lens),
                "flops": 4 * sum(lens) * case["hq"] * d}
    nq = sum(_lens(case["lens"], case["seed"]))
    nk = nq + sum(_lens(case["past"], case["seed"] + 1))
    return {"bytes": SIZE[case["dtype"]] * d * (2 * nq * case["hq"] + 2 * nk * hkv),
            "flops": 4 * _pairs(case) * case["hq"] * d}


# ------------------------------------------------------------------ inputs

def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape) -> torch.Tensor:
    return torch.randn(shape, generator=g, device="cuda")


def _spread(g, heads: int, d: int) -> torch.Tensor:
    """A size per channel of each head, a few of them large, as keys have them."""
    ch = torch.exp(0.4 * _randn(g, heads, d))
    return torch.where(torch.rand((heads, d), generator=g, device="cuda") < 1 / 64, 6 * ch, ch)


def _table(rot: int) -> torch.Tensor:
    """(position, frequency, (cos, sin)) of the usual base, made in 64 bits."""
    inv = 500000.0 ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)
    a = np.arange(TABLE, dtype=np.float64)[:, None] * inv
    return torch.from_numpy(np.stack([np.cos(a), np.sin(a)], axis=-1).astype(np.float32)).cuda()


def _slots(g, lens: list[int], page: int):
    """Pages in shuffled order: the table of each sequence and the slot of every token."""
    per = [max(1, math.ceil(n / page)) for n in lens]
    perm = torch.randperm(sum(per), generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(lens), max(per)), dtype=torch.int32, device="cuda")
    slots, at = [], 0
    for i, (n, p) in enumerate(zip(lens, per)):
        table[i, :p] = perm[at:at + p]
        t = torch.arange(n, device="cuda")
        slots.append(table[i, t // page].long() * page + t % page)
        at += p
    return table, torch.cat(slots), sum(per)


def _inputs(case, seed) -> dict:
    """The inputs, from the seed alone."""
    g = _gen(seed)
    kind, hkv, d = case["kind"], case["hkv"], case["d"]
    if kind == "rope":
        hq, n = case["hq"], case["tokens"]
        x = _randn(g, n, hq + 2 * hkv, d) * _spread(g, hq + 2 * hkv, d)
        # tokens of several sequences one after another, each somewhere in its text
        start = torch.randint(0, TABLE - n, (4,), generator=g, device="cuda")
        t = torch.arange(n, device="cuda")
        pos = (start[t * 4 // n] + t).to(torch.int32)
        w = [1 + 0.3 * _randn(g, d) if case["norm"] else None for _ in range(2)]
        return {"x": x.to(DT[case["src"]]).reshape(n, -1), "pos": pos, "table": _table(case["rot"]), "wq": w[0],
                "wk": w[1]}
    if kind == "kv":
        n = case["tokens"]
        pages = 2 * math.ceil(n / case["page"]) + 1
        if n <= 64:                          # one token of each sequence, anywhere in its page
            slots = torch.randperm(pages * case["page"], generator=g, device="cuda")[:n]
        else:
            perm = torch.randperm(pages, generator=g, device="cuda")
            t = torch.arange(n, device="cuda")
            slots = perm[t // case["page"]] * case["page"] + t % case["page"]
        k = (_randn(g, n, hkv, d) * _spread(g, hkv, d)).to(DT[case["src"]])
        v = (_randn(g, n, hkv, d) * (0.5 + torch.rand((hkv, d), generator=g, device="cuda"))).to(DT[case["src"]])
        return {"k": k, "v": v, "slots": slots, "pages": pages}
    hq = case["hq"]
    if kind == "decode":
        lens = _lens(case["lens"], case["seed"])
        table, slots, pages = _slots(g, lens, case["page"])
        total = sum(lens)
        ch = _spread(g, hkv, d)
        k = _randn(g, total, hkv, d) * ch
        v = _randn(g, total, hkv, d) * (0.5 + torch.rand((hkv, d), generator=g, device="cuda"))
        q = 2 * _randn(g, len(lens), hq, d) / ch.repeat_interleave(hq // hkv, 0)
        return {"k": k, "v": v, "q": q.to(DT[case["dtype"]]), "lens": lens, "table": table, "slots": slots,
                "pages": pages, "lens_dev": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    nq, past = _lens(case["lens"], case["seed"]), _lens(case["past"], case["seed"] + 1)
    nk = [a + b for a, b in zip(nq, past)]
    dt = DT[case["dtype"]]
    ch = _spread(g, hkv, d)
    cu = [torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32, device="cuda") for n in (nq, nk)]
    return {"q": (1.5 * _randn(g, sum(nq), hq, d) / ch.repeat_interleave(hq // hkv, 0)).to(dt),
            "k": (_randn(g, sum(nk), hkv, d) * ch).to(dt), "v": _randn(g, sum(nk), hkv, d).to(dt), "nq": nq, "nk": nk,
            "cu_q": cu[0], "cu_k": cu[1]}


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    kind = case["kind"]
    if own:
        if kind == "rope":
            dt, n = DT[case["out"]], case["tokens"]
            st["out"] = {p: torch.empty((n, h, case["d"]), dtype=dt, device="cuda")
                         for p, h in (("q", case["hq"]), ("k", case["hkv"]), ("v", case["hkv"]))}
        elif kind in ("kv", "decode"):
            from flatrun_amd.attention import KVCache4

            st["cache"] = c = KVCache4(st["pages"], case["page"], case["hkv"], case["d"])
            if kind == "decode":             # what earlier steps left in the cache
                c.write(st.pop("k"), st.pop("v"), st["slots"], st["slots"].numel(), dtype="f32",
                        stream=torch.cuda.current_stream())
                st["out"] = torch.empty_like(st["q"])
            else:
                st["out"] = {p: torch.empty(st["k"].shape, dtype=DT[case["out"]], device="cuda") for p in "kv"}
        else:
            st["out"] = torch.empty_like(st["q"])
        torch.cuda.synchronize()             # the inputs are there, whatever stream reads them
    elif kind in ("kv", "decode"):
        n = st["pages"] * case["page"]
        for p in "kv":
            st[p + "c"] = torch.zeros((n, case["hkv"], case["d"] // 2), dtype=torch.uint8, device="cuda")
            st[p + "d"] = torch.zeros((n, case["hkv"], case["d"] // BLOCK), dtype=torch.float16, device="cuda")
        if kind == "decode":
            for p in "kv":
                x = st.pop(p)
                for i in range(0, x.shape[0], 1 << 16):
                    _store(st, p, x[i:i + (1 << 16)], st["slots"][i:i + (1 << 16)])
    return st


# -------------------------------------------------------------- plain forms

def _store(st, p: str, x: torch.Tensor, slots: torch.Tensor) -> None:
    x = x.float().view(x.shape[0], x.shape[1], -1, BLOCK)
    e = x.gather(-1, x.abs().argmax(-1, keepdim=True))
    d = (e / -8).clamp(-65504, 65504).half()
    f = d.float()
    code = torch.where(f == 0, 8.0, (torch.round(x / f) + 8).clamp(0, 15)).to(torch.uint8)
    st[p + "c"][slots] = (code[..., 0::2] | (code[..., 1::2] << 4)).view(x.shape[0], x.shape[1], -1)
    st[p + "d"][slots] = d[..., 0]


def _load(st, p: str, slots: torch.Tensor) -> torch.Tensor:
    c = st[p + "c"][slots]
    code = torch.stack([c & 15, c >> 4], dim=-1).float().view(c.shape[0], c.shape[1], -1, BLOCK) - 8
    return (code * st[p + "d"][slots].float()[..., None]).view(c.shape[0], c.shape[1], -1)


def _rope_plain(st) -> list:
    case = st["case"]
    n, hq, hkv, d, rot = case["tokens"], case["hq"], case["hkv"], case["d"], case["rot"]
    x = st["x"].float().view(n, hq + 2 * hkv, d)
    cs = st["table"][st["pos"].long()][:, None]
    c, s = cs[..., 0], cs[..., 1]
    outs = []
    for y, w in ((x[:, :hq], st["wq"]), (x[:, hq:hq + hkv], st["wk"])):
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w
        r, rest = y[..., :rot], y[..., rot:]
        if case["pairs"] == "half":
            a, b = r[..., :rot // 2], r[..., rot // 2:]
            r = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
        else:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
        outs.append(torch.cat([r, rest], dim=-1))
    outs.append(x[:, hq + hkv:])
    return [y.to(DT[case["out"]]) for y in outs]


def _softmax_rows(s: torch.Tensor) -> torch.Tensor:
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _decode_plain(st) -> torch.Tensor:
    case = st["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    out = torch.zeros((len(st["lens"]), hq, d), device="cuda")
    at = 0
    for i, n in enumerate(st["lens"]):
        slots = st["slots"][at:at + n]
        at += n
        if n == 0:
            continue
        k = _load(st, "k", slots).permute(1, 2, 0).contiguous()                  # hkv, d, n
        v = _load(st, "v", slots).transpose(0, 1).contiguous()                   # hkv, n, d
        q = st["q"][i].float().view(hkv, hq // hkv, d)
        p = _softmax_rows(torch.matmul(q, k) * (1 / math.sqrt(d)))
        out[i] = torch.matmul(p, v).view(hq, d)
    return out.to(DT[case["dtype"]])


def _prefill_plain(st) -> torch.Tensor:
    case = st["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    g = hq // hkv
    out = torch.zeros(st["q"].shape, device="cuda")
    aq = ak = 0
    for nq, nk in zip(st["nq"], st["nk"]):
        kt = st["k"][ak:ak + nk].float().permute(1, 2, 0).contiguous()           # hkv, d, nk
        v = st["v"][ak:ak + nk].float().transpose(0, 1).contiguous()             # hkv, nk, d
        j = torch.arange(nk, device="cuda")
        for i in range(0, nq, 512):
            m = min(512, nq - i)
            last = min(nk, nk - nq + i + m) if case["causal"] else nk
            q = st["q"][aq + i:aq + i + m].float().view(m, hkv, g, d).permute(1, 2, 0, 3).reshape(hkv, g * m, d)
            s = torch.matmul(q, kt[:, :, :last].contiguous()) * (1 / math.sqrt(d))
            if case["causal"]:
                keep = j[:last] <= (nk - nq + i + torch.arange(m, device="cuda"))[:, None]
                s = s.view(hkv, g, m, last).masked_fill(~keep, float("-inf")).view(hkv, g * m, last)
            o = torch.matmul(_softmax_rows(s), v[:, :last].contiguous())
            out[aq + i:aq + i + m] = o.view(hkv, g, m, d).permute(2, 0, 1, 3).reshape(m, hq, d)
        aq, ak = aq + nq, ak + nk
    return out.to(DT[case["dtype"]])


# -------------------------------------------------------------------- passes

def run(st):
    case = st["case"]
    kind = case["kind"]
    if not own:
        if kind == "rope":
            return _rope_plain(st)
        if kind == "decode":
            return _decode_plain(st)
        if kind == "prefill":
            return _prefill_plain(st)
        for p in "kv":
            _store(st, p, st[p], st["slots"])
        return [_load(st, p, st["slots"]).to(DT[case["out"]]) for p in "kv"]
    from flatrun_amd import device

    s = torch.cuda.current_stream()
    if kind == "rope":
        o = st["out"]
        device.qk_norm_rope(st["x"], o["q"], o["k"], o["v"], case["tokens"], case["hq"], case["hkv"], case["d"],
                            st["table"], st["pos"], rot=case["rot"], interleaved=case["pairs"] == "interleaved",
                            q_norm=st["wq"], k_norm=st["wk"], eps=EPS, x_dtype=case["src"], out_dtype=case["out"],
                            stream=s)
        return [o["q"], o["k"], o["v"]]
    if kind == "kv":
        o = st["out"]
        st["cache"].write(st["k"], st["v"], st["slots"], case["tokens"], dtype=case["src"], stream=s)
        st["cache"].read(o["k"], o["v"], st["slots"], case["tokens"], dtype=case["out"], stream=s)
        return [o["k"], o["v"]]
    if kind == "decode":
        device.attn_decode(st["q"], st["cache"], st["table"], st["lens_dev"], st["out"], len(st["lens"]), case["hq"],
                           max_len=max(st["lens"]), dtype=case["dtype"], stream=s)
        return st["out"]
    device.attn_prefill(st["q"], st["k"], st["v"], st["out"], st["cu_q"], st["cu_k"], len(st["nq"]), sum(st["nq"]),
                        sum(st["nk"]), case["hq"], case["hkv"], case["d"], max_q=max(st["nq"]), max_k=max(st["nk"]),
                        causal=case["causal"], dtype=case["dtype"], stream=s)
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


def exact(case, seed):
    st = _inputs(case, seed)
    kind, hkv, d = case["kind"], case["hkv"], case["d"]
    if kind == "rope":
        n, hq, rot = case["tokens"], case["hq"], case["rot"]
        turn = torch.view_as_complex(st["table"][st["pos"].long()].double().contiguous())[:, None, :]
        x = st["x"].double().view(n, hq + 2 * hkv, d)
        out = []
        for lo, hi, w in ((0, hq, st["wq"]), (hq, hq + hkv, st["wk"])):
            y = x[:, lo:hi]
            if w is not None:
                y = w.double() * y / torch.sqrt(y.square().sum(-1, keepdim=True) / d + EPS)
            y = y.clone()
            if case["pairs"] == "half":
                z = torch.complex(y[..., :rot // 2].contiguous(), y[..., rot // 2:rot].contiguous()) * turn
                y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
            else:
                z = torch.complex(y[..., 0:rot:2].contiguous(), y[..., 1:rot:2].contiguous()) * turn
                y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
            out.append(y)
        return out + [x[:, hq + hkv:]]
    if kind == "kv":
        return [_block_values(st["k"]), _block_values(st["v"])]
    hq = case["hq"]
    g = hq // hkv
    if kind == "decode":
        k, v = (torch.cat([_block_values(x) for x in st[p].split(1 << 15)]) for p in "kv")
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        at = 0
        for i, n in enumerate(st["lens"]):
            for h in range(hq if n else 0):
                s = (k[at:at + n, h // g] * st["q"][i, h].double()).sum(-1) / math.sqrt(d)
                out[i, h] = (torch.exp(s - torch.logsumexp(s, 0))[:, None] * v[at:at + n, h // g]).sum(0)
            at += n
        return out
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    aq = ak = 0
    for nq, nk in zip(st["nq"], st["nk"]):
        rows = torch.arange(nk - nq, nk, device="cuda")
        for h in range(hq):
            k, v = st["k"][ak:ak + nk, h // g].double(), st["v"][ak:ak + nk, h // g].double()
            for i in range(0, nq, 4096):
                r = slice(i, min(nq, i + 4096))
                s = st["q"][aq:aq + nq, h][r].double() @ k.t().contiguous() / math.sqrt(d)
                if case["causal"]:
                    s = torch.where(torch.arange(nk, device="cuda") > rows[r][:, None], float("-inf"), s)
                out[aq:aq + nq, h][r] = torch.exp(s - torch.logsumexp(s, -1, keepdim=True)) @ v
        aq, ak = aq + nq, ak + nk
    return out
