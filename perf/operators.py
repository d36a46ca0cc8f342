"""Measured cases of the operators of one batched serving step over a paged K/V cache.

  append   keys and values of new tokens into a paged cache, rotated on the way, with their queries
  attend   one new token of each sequence against its cached keys and values
  rules    penalties for repeated tokens, biases and grammar masks on logits, and the greedy id

`own = False` computes them from elementary torch operations in 32 bits; `own = True` through the
kq package. Lengths, positions and counts follow from a case alone, all values from the seed."""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
E4M3_MAX = 448.0


def kq():
    package = os.path.join(ROOT, "oxcoder-9b_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import kq as module
    return module


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # the decode step of one sequence of the default model (32 query, 8 K/V heads): pure latency
        {"name": "append-one", "op": "append", "n": 1, "seqs": 1, "heads": 32, "kv": 8, "hd": 128, "rot": 128,
         "page": 64, "ctx": 4096, "src": "f32", "cache": "f16"},
        # a full batched step into an 8-bit cache of short pages
        {"name": "append-128-8bit", "op": "append", "n": 128, "seqs": 128, "heads": 32, "kv": 8, "hd": 128, "rot": 128,
         "page": 16, "ctx": 4096, "src": "bf16", "cache": "e4m3"},
        # chunks of several prompts in one call, wide heads of which a quarter turns
        {"name": "append-chunks-wide", "op": "append", "n": 1021, "seqs": 5, "heads": 16, "kv": 4, "hd": 256, "rot": 64,
         "page": 32, "ctx": 32768, "src": "f32", "cache": "f16"},
        # one long prompt of 16-bit activations
        {"name": "append-prompt", "op": "append", "n": 8192, "seqs": 3, "heads": 32, "kv": 8, "hd": 128, "rot": 128,
         "page": 64, "ctx": 32768, "src": "bf16", "cache": "bf16"},
        # batch-1 decode at context 4K, the default model's layer
        {"name": "attend-one-4k", "op": "attend", "n": 1, "heads": 32, "kv": 8, "hd": 128, "page": 64, "least": 4096,
         "most": 4096, "empty": 0, "window": 0, "q": "f32", "cache": "f16"},
        # a full batched step, conversations from a few tokens to the whole context
        {"name": "attend-128-ragged", "op": "attend", "n": 128, "heads": 32, "kv": 8, "hd": 128, "page": 16, "least": 9,
         "most": 4096, "empty": 0, "window": 0, "q": "f32", "cache": "f16"},
        # 64 sequences of contexts up to 32K
        {"name": "attend-64-32k", "op": "attend", "n": 64, "heads": 32, "kv": 8, "hd": 128, "page": 64, "least": 8192,
         "most": 32768, "empty": 0, "window": 0, "q": "f16", "cache": "f16"},
        # few very long documents in an 8-bit cache, wide heads
        {"name": "attend-3-128k-8bit", "op": "attend", "n": 3, "heads": 16, "kv": 4, "hd": 256, "page": 32,
         "least": 100000, "most": 131072, "empty": 0, "window": 0, "q": "bf16", "cache": "e4m3"},
        # a head of its own for each query, a sliding window, odd lengths and slots that hold nothing yet
        {"name": "attend-37-window", "op": "attend", "n": 37, "heads": 12, "kv": 12, "hd": 64, "page": 16, "least": 1,
         "most": 5001, "empty": 4, "window": 500, "q": "bf16", "cache": "bf16"},
        # one sequence's next token over the default vocabulary
        {"name": "rules-one", "op": "rules", "n": 1, "vocab": 151936, "hist": 700, "bias": 16, "masks": 1, "type": "f32"},
        # a full batched step: long histories, biases, a grammar for most rows
        {"name": "rules-128", "op": "rules", "n": 128, "vocab": 151936, "hist": 4096, "bias": 300, "masks": 9, "type": "f32"},
        # a small odd vocabulary in 16 bits
        {"name": "rules-45-odd", "op": "rules", "n": 45, "vocab": 32003, "hist": 1500, "bias": 40, "masks": 45, "type": "bf16"},
    ]


def _log(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "rules"])
    if op == "rules":
        vocab = _log(rng, 4096, 160000)
        n = min(_log(rng, 1, 256), max(1, 120 * 151936 // vocab))
        return {"op": op, "n": n, "vocab": vocab, "hist": _log(rng, 1, 6000), "bias": rng.choice([0, 1, 17, 300]),
                "masks": rng.choice([0, 1, max(1, n // 2), n]), "type": rng.choice(["f32", "f32", "bf16", "f16"])}
    hd = rng.choice([64, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8, 12])
    heads = kv * rng.choice([1, 2, 3, 4, 7, 8, 12])
    page = rng.choice([16, 32, 64, 128])
    cache = rng.choice(["f16", "bf16", "e4m3"])
    if op == "append":
        n = _log(rng, 1, max(64, min(8192, 3500 * 48 * 128 // ((heads + 2 * kv) * hd))))
        if cache == "e4m3":
            n = min(n, 3000000 // (kv * hd) // 2)
        return {"op": op, "n": n, "seqs": rng.randint(1, min(n, 128)), "heads": heads, "kv": kv, "hd": hd,
                "rot": rng.choice([hd, hd, hd // 2, hd // 4]), "page": page, "ctx": rng.choice([16384, 32768, 131072]),
                "src": rng.choice(["f32", "f16", "bf16"]), "cache": cache}
    n = _log(rng, 1, 200)
    most = _log(rng, 1, max(64, min(131072, 60 * 20000 * 1024 // (n * kv * hd))))
    q = rng.choice(["f32", cache if cache != "e4m3" else "f16"])
    return {"op": op, "n": n, "heads": heads, "kv": kv, "hd": hd, "page": page, "least": max(1, most // rng.choice([1, 8, 200])),
            "most": most, "empty": rng.choice([0, 0, 1]) if n > 1 else 0, "window": rng.choice([0, 0, 0, 300]), "q": q,
            "cache": cache}


def spread(n, least, most, empty):
    """n lengths between least and most, even over the logarithm; every (n // empty)-th is 0."""
    rng = random.Random("%d %d %d" % (n, least, most))
    got = [_log(rng, least, most) for _ in range(n)]
    for j in range(empty):
        got[(2 * j + 1) * n // (2 * empty)] = 0
    return got


def places(c):
    """(row of the page table, position) of each new token: consecutive positions of each sequence."""
    rng = random.Random("%d %d %d" % (c["n"], c["seqs"], c["ctx"]))
    cuts = sorted(rng.sample(range(1, c["n"]), c["seqs"] - 1)) if c["seqs"] > 1 else []
    seq, pos = [], []
    for s, (a, b) in enumerate(zip([0] + cuts, cuts + [c["n"]])):
        start = rng.randint(0, c["ctx"] - (b - a))
        seq += [s] * (b - a)
        pos += range(start, start + b - a)
    return seq, pos


def histories(c):
    rng = random.Random("%d %d %d" % (c["n"], c["vocab"], c["hist"]))
    length = [_log(rng, max(1, c["hist"] // 64), c["hist"]) for _ in range(c["n"])]
    return length, [rng.randint(0, v) for v in length]


# ----------------------------------------------------------------------------- inputs
def _normal(g, shape, kind, scale=1.0):
    x = torch.empty(shape, device="cuda", dtype=torch.float16 if kind == "e4m3" else TYPES[kind])
    x.normal_(0.0, scale, generator=g)
    return x.to(TYPES[kind]) if kind == "e4m3" else x


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _ints(v, kind=torch.int32):
    return torch.tensor(v, dtype=kind, device="cuda")


def _pool(c, g, pages):
    """K and V pages [page][kv head][row][dim] and their scales, and the pages in random order."""
    shape = (pages, c["kv"], c["page"], c["hd"])
    s = {"k": _normal(g, shape, c["cache"]), "v": _normal(g, shape, c["cache"]), "ks": None, "vs": None}
    if c["cache"] == "e4m3":
        s["ks"] = torch.rand(c["kv"], device="cuda", generator=g) * 0.02 + 0.03
        s["vs"] = torch.rand(c["kv"], device="cuda", generator=g) * 0.02 + 0.03
        for name in ("k", "v"):  # values that use the format's range
            s[name] = (s[name].to(torch.float16) * 24).to(torch.float8_e4m3fn)
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    return s, order


def prepare(case, seed):
    c, g = case, _generator(seed)
    if c["op"] == "rules":
        s = _prepare_rules(c, g)
    elif c["op"] == "append":
        s = _prepare_append(c, g)
    else:
        s = _prepare_attend(c, g)
    s["case"] = c
    if own and c["op"] != "rules":
        s["cache"] = kq().PagedCache(s["k"], s["v"], k_scale=s["ks"], v_scale=s["vs"])
    return s


def _prepare_append(c, g):
    seq, pos = places(c)
    held = {}  # the pages that the new tokens fall into, numbered as they come
    for a, p in zip(seq, pos):
        held.setdefault((a, p // c["page"]), len(held))
    wide = c["ctx"] // c["page"]
    pages = len(held) + 3
    s, order = _pool(c, g, pages)
    table = torch.zeros((c["seqs"], wide), dtype=torch.int32, device="cuda")
    at = torch.tensor(list(held), device="cuda")
    table[at[:, 0], at[:, 1]] = order[:len(held)]
    n = c["n"]
    width = (c["heads"] + 2 * c["kv"]) * c["hd"]  # one projection's rows: queries, keys, values
    rows = _normal(g, (n, width), c["src"])
    q, k, v = (t.view(n, -1, c["hd"]) for t in rows.split([c["heads"] * c["hd"], c["kv"] * c["hd"], c["kv"] * c["hd"]], 1))
    half = c["rot"] // 2
    inv = 1e6 ** (-2.0 * np.arange(half) / c["rot"])
    angle = torch.arange(c["ctx"], device="cuda", dtype=torch.float64)[:, None] * torch.tensor(inv, device="cuda")
    s.update(table=table, seq=_ints(seq), pos=_ints(pos), q_new=q, k_new=k, v_new=v, cos=angle.cos().float(),
             sin=angle.sin().float(), q_out=torch.empty((n, c["heads"], c["hd"]), dtype=TYPES[c["src"]], device="cuda"))
    return s


def _prepare_attend(c, g):
    lens = spread(c["n"], c["least"], c["most"], c["empty"])
    each = [-(-v // c["page"]) for v in lens]
    wide = max(each + [1])
    s, order = _pool(c, g, sum(each) + 2)
    table = torch.zeros((c["n"], wide), dtype=torch.int32, device="cuda")
    own_pages = torch.arange(wide, device="cuda")[None, :] < _ints(each)[:, None]
    table[own_pages] = order[:sum(each)]
    q = _normal(g, (c["n"], c["heads"], c["hd"]), c["q"], 1.5)
    s.update(table=table, lens=_ints(lens), lens_host=lens, q=q, out=torch.empty_like(q))
    return s


def _prepare_rules(c, g):
    n, vocab = c["n"], c["vocab"]
    length, prompt = histories(c)
    u = torch.rand((n, max(length)), device="cuda", generator=g)
    hist = (u.pow(4) * vocab).to(torch.int32).clamp_(max=vocab - 1)  # few ids often, many seldom
    s = {"logits": _normal(g, (n, vocab), c["type"], 3.0), "hist": hist, "hist_len": _ints(length), "prompt_len": _ints(prompt),
         "rep": 1.0 + torch.rand(n, device="cuda", generator=g) * 0.4, "freq": torch.rand(n, device="cuda", generator=g) * 0.5,
         "pres": torch.rand(n, device="cuda", generator=g) - 0.3, "ids": None, "bias": None, "mask": None, "mask_row": None}
    if c["bias"]:
        picks = torch.rand((n, min(vocab, 8 * c["bias"])), device="cuda", generator=g).argsort(1)[:, :c["bias"]]
        ids = (picks * (vocab // (8 * c["bias"]) or 1)).to(torch.int32).contiguous()  # distinct ids
        ids[:, c["bias"] - c["bias"] // 4:] = -1  # rows are padded
        s["ids"], s["bias"] = ids, torch.randn((n, c["bias"]), device="cuda", generator=g) * 4
    if c["masks"]:
        words = (vocab + 31) // 32
        shape = (c["masks"], words)
        a, b, d = (torch.randint(-2**31, 2**31, shape, device="cuda", dtype=torch.int32, generator=g) for _ in range(3))
        few = torch.arange(c["masks"], device="cuda")[:, None] % 3 == 1
        s["mask"] = torch.where(few, a & b & d & a.roll(1, 1) & b.roll(1, 1), a | b)
        if c["masks"] > 4:
            s["mask"][4] = 0  # a grammar that has come to its end allows nothing
        row = [(-1 if i % 7 == 3 else i % c["masks"]) for i in range(n)]
        s["mask_row"] = _ints(row)
    s.update(out=torch.empty_like(s["logits"]), best=torch.empty(n, dtype=torch.int32, device="cuda"))
    return s


# ----------------------------------------------------------------------------- one pass
def run(state):
    s = state
    c = s["case"]
    if c["op"] == "append":
        return _append_own(s) if own else _append_plain(s)
    if c["op"] == "attend":
        return {"out": s["cache"].attend(s["q"], s["table"], s["lens"], s["out"], window=c["window"])} if own else _attend_plain(s)
    return _rules_own(s) if own else _rules_plain(s)


def _append_own(s):
    s["cache"].append(s["k_new"], s["v_new"], s["table"], s["pos"], seq=s["seq"], rope=(s["cos"], s["sin"]), q=s["q_new"],
                      q_out=s["q_out"])
    return {"k": s["k"], "v": s["v"], "q": s["q_out"]}


def _rules_own(s):
    kq().logit_rules(s["logits"], s["out"], best=s["best"], hist=s["hist"], hist_len=s["hist_len"], prompt_len=s["prompt_len"],
                     repetition=s["rep"], frequency=s["freq"], presence=s["pres"], bias_ids=s["ids"], bias=s["bias"],
                     mask=s["mask"], mask_row=s["mask_row"])
    return {"logits": s["out"], "best": s["best"]}


def _turn(x, cos, sin, rot):
    x = x.float()
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)


def _store(pool, where, x, scale):
    if scale is not None:
        x = (x / scale[None, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
    x = x.to(pool.dtype)
    if scale is not None:
        pool, x = pool.view(torch.uint8), x.view(torch.uint8)
    pool[where[0], :, where[1]] = x


def _append_plain(s):
    c = s["case"]
    pos, seq = s["pos"].long(), s["seq"].long()
    where = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
    cos, sin = s["cos"][pos][:, None, :], s["sin"][pos][:, None, :]
    _store(s["k"], where, _turn(s["k_new"], cos, sin, c["rot"]), s["ks"])
    _store(s["v"], where, s["v_new"].float(), s["vs"])
    return {"k": s["k"], "v": s["v"], "q": _turn(s["q_new"], cos, sin, c["rot"]).to(s["q_new"].dtype)}


def _first(length, window):
    return max(0, length - window) if window else 0


def _gather(pool, pages, first, length, page, scale):
    """[kv][keys][dim] in 32 bits."""
    x = pool[pages] if scale is None else pool.view(torch.uint8)[pages].view(pool.dtype)
    x = x.float().transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])
    base = first // page * page
    x = x[:, first - base:length - base]
    return x if scale is None else x * scale[:, None, None]


def _attend_plain(s):
    c = s["case"]
    out = torch.zeros_like(s["q"])
    group = c["heads"] // c["kv"]
    for i, length in enumerate(s["lens_host"]):
        if not length:
            continue
        first = _first(length, c["window"])
        pages = s["table"][i, first // c["page"]:-(-length // c["page"])].long()
        k = _gather(s["k"], pages, first, length, c["page"], s["ks"])
        v = _gather(s["v"], pages, first, length, c["page"], s["vs"])
        q = s["q"][i].float().view(c["kv"], group, c["hd"])
        z = (q @ k.transpose(1, 2)) * (1.0 / math.sqrt(c["hd"]))
        p = (z - z.amax(-1, keepdim=True)).exp()
        o = (p @ v) / p.sum(-1, keepdim=True)
        out[i] = o.view(c["heads"], c["hd"]).to(out.dtype)
    return {"out": out}


def _rules_plain(s):
    c = s["case"]
    n, vocab = c["n"], c["vocab"]
    z = s["logits"].float()
    at = torch.arange(s["hist"].shape[1], device="cuda")[None, :]
    used = at < s["hist_len"][:, None]
    answered = used & (at >= s["prompt_len"][:, None])
    hist = s["hist"].long()
    count = torch.zeros((n, vocab), dtype=torch.int32, device="cuda").scatter_add_(1, hist, answered.int())
    seen = torch.zeros((n, vocab), dtype=torch.int32, device="cuda").scatter_add_(1, hist, used.int()) > 0
    rep = s["rep"][:, None]
    z = torch.where(seen, torch.where(z > 0, z / rep, z * rep), z)
    z = z - (s["freq"][:, None] * count.float() + s["pres"][:, None] * (count > 0).float())
    if s["ids"] is not None:
        add = torch.zeros((n, vocab + 1), device="cuda")
        add.scatter_(1, torch.where(s["ids"] < 0, vocab, s["ids"]).long(), s["bias"])
        z = z + add[:, :vocab]
    if s["mask"] is not None:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        allowed = bits.view(bits.shape[0], -1)[:, :vocab].bool()[s["mask_row"].long().clamp(min=0)]
        allowed = allowed | (s["mask_row"] < 0)[:, None]
        z = torch.where(allowed, z, -math.inf)
    z = z.to(s["logits"].dtype)
    top = z.amax(1, keepdim=True)
    ids = torch.arange(vocab, device="cuda", dtype=torch.int32)[None, :]
    best = torch.where((z == top) & (z > -math.inf), ids, vocab).amin(1)
    return {"logits": z, "best": torch.where(best == vocab, -1, best).int()}


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "append":
        n, hd = c["n"], c["hd"]
        row = (c["heads"] + 2 * c["kv"]) * hd * SIZE[c["src"]]
        stored = 2 * c["kv"] * hd * SIZE[c["cache"]] + c["heads"] * hd * SIZE[c["src"]]
        return {"bytes": n * (row + stored + c["rot"] * 4 + 12), "flops": n * ((c["heads"] + c["kv"]) * c["rot"] * 3 + c["kv"] * hd * 2)}
    if c["op"] == "attend":
        keys = sum(v - _first(v, c["window"]) for v in spread(c["n"], c["least"], c["most"], c["empty"]))
        table = sum(-(-v // c["page"]) - _first(v, c["window"]) // c["page"] for v in spread(c["n"], c["least"], c["most"], c["empty"]))
        return {"bytes": keys * 2 * c["kv"] * c["hd"] * SIZE[c["cache"]] + 2 * c["n"] * c["heads"] * c["hd"] * SIZE[c["q"]] + 4 * table,
                "flops": keys * c["heads"] * c["hd"] * 4}
    n, vocab = c["n"], c["vocab"]
    small = 4 * sum(histories(c)[0]) + n * (8 * c["bias"] + 28) + c["masks"] * ((vocab + 31) // 32) * 4
    return {"bytes": 2 * n * vocab * SIZE[c["type"]] + small, "flops": 6 * n * vocab}


# ----------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] == "append":
        return _exact_append(s, c)
    if c["op"] == "attend":
        return _exact_attend(s, c)
    return _exact_rules(s, c)


def _exact_append(s, c):
    """Every pair turned as a complex number."""
    half = c["rot"] // 2
    seq, pos = places(c)
    out = {}
    unit = torch.complex(s["cos"].double(), s["sin"].double())[torch.tensor(pos, device="cuda")]
    for name in ("q", "k"):
        x = s[name + "_new"].double().clone()
        turned = torch.complex(x[:, :, :half], x[:, :, half:c["rot"]]) * unit.unsqueeze(1)
        x[:, :, :half], x[:, :, half:c["rot"]] = turned.real, turned.imag
        out[name] = x
    table = s["table"].cpu().numpy()
    page = np.array([table[a, p // c["page"]] for a, p in zip(seq, pos)], dtype=np.int64)
    rows = torch.tensor(page * c["page"] + np.array(pos) % c["page"], device="cuda")
    for name, x, scale in (("k", out["k"], s["ks"]), ("v", s["v_new"].double(), s["vs"])):
        if scale is not None:
            x = x / scale.double().view(1, -1, 1)
        pool = s[name].double().permute(0, 2, 1, 3).reshape(-1, c["kv"], c["hd"])
        pool[rows] = x
        out[name] = pool.view(-1, c["page"], c["kv"], c["hd"]).permute(0, 2, 1, 3).contiguous()
    return out


def _exact_attend(s, c):
    """A head at a time: log-sum-exp weights over the gathered keys."""
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = c["heads"] // c["kv"]
    for i, length in enumerate(s["lens_host"]):
        first = _first(length, c["window"])
        if length <= first:
            continue
        t = torch.arange(first, length, device="cuda")
        page, row = s["table"][i].long()[t // c["page"]], t % c["page"]
        for g in range(c["kv"]):
            if s["ks"] is None:
                k, v = s["k"][page, g, row].double(), s["v"][page, g, row].double()
            else:
                k = s["k"].view(torch.uint8)[page, g, row].view(torch.float8_e4m3fn).double() * s["ks"][g].double()
                v = s["v"].view(torch.uint8)[page, g, row].view(torch.float8_e4m3fn).double() * s["vs"][g].double()
            z = torch.einsum("td,hd->ht", k, s["q"][i, g * group:(g + 1) * group].double()) / c["hd"] ** 0.5
            out[i, g * group:(g + 1) * group] = torch.einsum("ht,td->hd", torch.exp(z - torch.logsumexp(z, 1, keepdim=True)), v)
    return {"out": out}


def _exact_rules(s, c):
    """Row by row, over the ids that occur."""
    z = s["logits"].double()
    hist, ids = s["hist"].cpu().numpy(), None if s["ids"] is None else s["ids"].cpu().numpy()
    length, prompt = histories(c)
    for i in range(c["n"]):
        occur, count = np.unique(hist[i, :length[i]], return_counts=True)
        late, late_count = np.unique(hist[i, min(prompt[i], length[i]):length[i]], return_counts=True)
        rep, freq, pres = (float(s[k][i]) for k in ("rep", "freq", "pres"))
        at = torch.tensor(occur, device="cuda").long()
        v = z[i, at]
        z[i, at] = torch.where(v > 0, v / rep, v * rep)
        at = torch.tensor(late, device="cuda").long()
        z[i, at] -= freq * torch.tensor(late_count, device="cuda").double() + pres
        if ids is not None:
            keep = ids[i] >= 0
            z[i, torch.tensor(ids[i][keep], device="cuda").long()] += s["bias"][i].double()[torch.tensor(keep, device="cuda")]
    if s["mask"] is not None:
        word = s["mask"].cpu().numpy().view(np.uint8)
        allowed = np.unpackbits(word, axis=1, bitorder="little")[:, :c["vocab"]].astype(bool)
        for i, r in enumerate(s["mask_row"].tolist()):
            if r >= 0:
                z[i, torch.tensor(~allowed[r], device="cuda")] = -math.inf
    return {"logits": z, "best": None}
