"""The operators of a serving step over a paged cache, as cases that can be timed and checked.

A program that serves several sequences from one pool of memory does, in every layer of a step: it turns queries and keys by their
positions (rotate), writes the new rows of keys and values to the pages of their sequences (store; a pool's rows also come back, when a
sequence moves or is inspected: load), lets the new tokens attend to all that their sequences hold (attend), and where tokens were drafted
by a smaller model, finds out at the step's end how many of them stand (verify).

Head layouts are those of this repository's models: 32 and 40 heads of 128 with as many key heads (7B, 13B), 32 over 8 and 16 over 4
(block models of width 4096 and 2048), 4 of 64 (the tiny one); vocabularies 32000 and 128256.

The pool is bytes, in the layout that include/llava_hip.h gives it (lv_paged_cache); prepare() fills it by that description.  Without `own`,
run() is elementary torch operations in 32 bits: 64 for angles, and for the sums a random number is compared with.
"""
import importlib
import math

import numpy as np
import torch

own = False

PAIRS = {"neighbours": 0, "halves": 1}
FLOATS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CACHES = ("f16", "bf16", "q8_0", "q4_0")
HEADS = ((32, 32, 128), (40, 40, 128), (32, 8, 128), (16, 4, 128), (4, 4, 64))
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # the smallest call: one chat, its next token behind a short context, 32-bit activations over the 7B layer's fp16 rows
        dict(name="attend, 1 token behind 510", kind="attend", heads=32, kv_heads=32, dim=128, cache="f16", type="f32", page=16, seqs=1, len=511, new=1, mix=False, ragged=False,
             window=0, sinks=False),
        # a server's step: 64 chats of different lengths, 8-bit rows, grouped heads
        dict(name="attend, 64 chats, 8 bits", kind="attend", heads=32, kv_heads=8, dim=128, cache="q8_0", type="bf16", page=64, seqs=64, len=8190, new=1, mix=False, ragged=True,
             window=0, sinks=False),
        # one chat behind a very long document: few rows, a long axis
        dict(name="attend, 1 token, long document", kind="attend", heads=32, kv_heads=8, dim=128, cache="f16", type="f16", page=128, seqs=1, len=131072, new=1, mix=False,
             ragged=False, window=0, sinks=False),
        # up to five drafted tokens of each of 16 chats at once, 4-bit rows, a learned logit a head
        dict(name="attend, drafts of 16 chats", kind="attend", heads=16, kv_heads=4, dim=128, cache="q4_0", type="f16", page=32, seqs=16, len=3001, new=5, mix=False, ragged=True,
             window=0, sinks=True),
        # a chunk of a long prompt: the largest call, bound by arithmetic
        dict(name="attend, 2048 behind 6144", kind="attend", heads=32, kv_heads=8, dim=128, cache="bf16", type="bf16", page=64, seqs=1, len=8192, new=2048, mix=False, ragged=False,
             window=0, sinks=False),
        # the new rows of 64 chats, 8-bit
        dict(name="store, 64 chats, 8 bits", kind="store", kv_heads=8, dim=128, cache="q8_0", type="bf16", page=64, seqs=64, len=4000, new=1, ragged=True),
        # a long prompt's rows, 4-bit, from 32-bit projections
        dict(name="store, 4095 tokens, 4 bits", kind="store", kv_heads=32, dim=128, cache="q4_0", type="f32", page=32, seqs=1, len=4500, new=4095, ragged=False),
        # all rows of four sequences, to be moved elsewhere
        dict(name="load, 4 sequences, 8 bits", kind="load", kv_heads=8, dim=128, cache="q8_0", type="f16", page=16, seqs=4, len=16001, ragged=True),
        # one token's queries and keys of a 7B layer
        dict(name="rotate, 1 token", kind="rotate", tokens=1, heads=64, dim=128, rot=128, type="f32", pairs="neighbours", axes=1, base=10000.0),
        # a prompt with pictures: queries and keys, positions in time, height and width
        dict(name="rotate, 6001 tokens, 3 axes", kind="rotate", tokens=6001, heads=40, dim=128, rot=128, type="bf16", pairs="halves", axes=3, base=1000000.0),
        # one chat's four drafts
        dict(name="verify, 1 chat", kind="verify", seqs=1, drafts=4, vocab=32000, ragged=False, sampled=True, near=0.8),
        # a server's drafts
        dict(name="verify, 48 chats", kind="verify", seqs=48, drafts=7, vocab=128256, ragged=True, sampled=True, near=0.9),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "store", "load", "rotate", "verify"))
    heads, kv_heads, dim = rng.choice(HEADS)
    c = dict(kind=kind)
    if kind == "attend":
        new = rng.choice((1, 1, _log(rng, 2, 16), _log(rng, 17, 1500)))
        seqs = _log(rng, 1, 64) if new < 17 else _log(rng, 1, 6)
        most = min(100000, 2 * 10 ** 8 // (seqs * kv_heads * dim), 10 ** 11 // (4 * dim * heads * new * seqs))
        c.update(heads=heads, kv_heads=kv_heads, dim=dim, cache=rng.choice(CACHES), type=rng.choice(("f32", "f16", "bf16")), page=rng.choice((16, 32, 64, 128, 256)), seqs=seqs,
                 len=_log(rng, new, max(new, most)), new=new, mix=new > 16 and rng.random() < 0.4, ragged=rng.random() < 0.6, window=rng.choice((0, 0, _log(rng, 8, 4096))),
                 sinks=rng.random() < 0.3)
    elif kind == "store":
        seqs = _log(rng, 1, 64)
        new = rng.choice((1, _log(rng, 2, max(2, 4000 // seqs))))
        c.update(kv_heads=kv_heads, dim=dim, cache=rng.choice(CACHES), type=rng.choice(("f32", "f16", "bf16")), page=rng.choice((16, 32, 64, 128, 256)), seqs=seqs,
                 len=new + _log(rng, 1, 4000), new=new, ragged=rng.random() < 0.5)
    elif kind == "load":
        seqs = _log(rng, 1, 16)
        c.update(kv_heads=kv_heads, dim=dim, cache=rng.choice(CACHES), type=rng.choice(("f32", "f16", "bf16")), page=rng.choice((16, 32, 64, 128, 256)), seqs=seqs,
                 len=_log(rng, 1, 60000 // seqs), ragged=rng.random() < 0.5)
    elif kind == "rotate":
        c.update(tokens=_log(rng, 1, 8000), heads=rng.choice((heads, heads + kv_heads)), dim=dim, rot=rng.choice((dim, dim, dim // 2)), type=rng.choice(("f32", "f16", "bf16")),
                 pairs=rng.choice(("neighbours", "halves")), axes=rng.choice((1, 2, 3)), base=rng.choice((10000.0, 500000.0, 1000000.0)))
    else:
        c.update(seqs=_log(rng, 1, 48), drafts=rng.randint(1, 8), vocab=rng.choice((512, 32000, 32000, 128256)), ragged=rng.random() < 0.5, sampled=rng.random() < 0.7,
                 near=rng.choice((0.3, 0.6, 0.9, 0.97)))
    return c


# ---- sizes of a case, the same for every seed --------------------------------------------------------------------------------

def _lengths(c):
    """tokens of each sequence, and how many of them are new (of each one's end)"""
    b = np.arange(c["seqs"])
    new = np.full(c["seqs"], c.get("new", 0))
    if c.get("mix"):
        new[1:] = 1
    lens = np.full(c["seqs"], c["len"])
    if c["ragged"]:
        lens = lens - (b * 7919) % max(1, c["len"] // 2 + 1)
        if c.get("new", 0) > 1 and not c.get("mix"):
            new = 1 + (new - 1 + b * 31) % new
    if c["kind"] == "load":
        new = lens
    return np.maximum(lens, new), new


def _row_bytes(c):
    """codes and scales of one head's row"""
    d = c["dim"]
    return {"f16": (2 * d, 0), "bf16": (2 * d, 0), "q8_0": (d, d // 16), "q4_0": (d // 2, d // 16)}[c["cache"]]


def work(c):
    kind = c["kind"]
    if kind == "rotate":
        n = c["tokens"] * c["heads"] * c["dim"]
        return {"bytes": 2 * n * SIZE[c["type"]] + 4 * c["axes"] * c["tokens"], "flops": 3 * c["tokens"] * c["heads"] * c["rot"]}
    if kind == "verify":
        return {"bytes": c["seqs"] * (c["vocab"] * 4 * (2 if c["sampled"] else 1) + 8 * c["drafts"] * 4), "flops": 3 * c["seqs"] * c["vocab"]}
    lens, new = _lengths(c)
    row = 2 * c["kv_heads"] * sum(_row_bytes(c))
    if kind == "store":       # written, and read again
        return {"bytes": int(new.sum()) * (2 * row + 2 * 2 * c["kv_heads"] * c["dim"] * SIZE[c["type"]]), "flops": 8 * int(new.sum()) * c["kv_heads"] * c["dim"]}
    if kind == "load":
        return {"bytes": int(new.sum()) * (row + 2 * c["kv_heads"] * c["dim"] * SIZE[c["type"]]), "flops": 2 * int(new.sum()) * c["kv_heads"] * c["dim"]}
    w = c["window"] or 1 << 40
    seen = pairs = 0
    for n, m in zip(lens.tolist(), new.tolist()):
        seen += min(n, m - 1 + w)
        # row i of m sees min(n - m + i + 1, w) keys
        full = max(0, min(m, n - w))      # rows that see a whole window
        pairs += full * w + sum(range(n - m + 1, n - full + 1)) if full < m else m * w
    return {"bytes": seen * row + 2 * int(new.sum()) * c["heads"] * c["dim"] * SIZE[c["type"]], "flops": 4 * c["dim"] * c["heads"] * pairs}


# ---- inputs -------------------------------------------------------------------------------------------------------------------

def _part(c, pool, which):
    """(codes, scales) of the keys (0) or the values (1), as views of the pool: [page][kv head][token][...]"""
    cb, sb = _row_bytes(c)
    page = c["page"]
    at = which * page * (cb + sb)
    kind = {"f16": torch.float16, "bf16": torch.bfloat16, "q8_0": torch.int8, "q4_0": torch.uint8}[c["cache"]]
    codes, scales = pool[:, :, at:at + page * cb], pool[:, :, at + page * cb:at + page * (cb + sb)]
    return codes.view(kind).unflatten(-1, (page, -1)), scales.view(torch.float16).unflatten(-1, (page, -1)) if sb else None


def _parts(c, pool):
    return _part(c, pool, 0), _part(c, pool, 1)


def _fill(c, g, codes, scales):
    """rows as a model leaves them: numbers of about 1"""
    dev = codes.device
    if scales is None:
        codes.copy_(torch.randn(codes.shape, generator=g, device=dev, dtype=torch.float32))
        return
    four = c["cache"] == "q4_0"
    codes.copy_(torch.randint(0 if four else -127, 256 if four else 128, codes.shape, generator=g, device=dev, dtype=torch.int16))
    d = (0.5 + torch.rand(scales.shape, generator=g, device=dev)) / (4.6 if four else 73)
    scales.copy_(d * torch.where(torch.rand(scales.shape, generator=g, device=dev) < 0.5, -1.0, 1.0) if four else d)


def _pool(c, g, dev):
    """a pool with rows in all of its pages, and which page holds what of each sequence: a page more than the longest one needs, pages in no order"""
    lens, new = _lengths(c)
    per = (int(lens.max()) + c["page"] - 1) // c["page"] + 1
    need = (lens + c["page"] - 1) // c["page"]
    pages = int(need.sum()) + 3
    size = 2 * c["page"] * sum(_row_bytes(c))
    pool = torch.empty(pages, c["kv_heads"], size, dtype=torch.uint8, device=dev)
    _fill(c, g, *_part(c, pool, 0))
    _fill(c, g, *_part(c, pool, 1))
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(c["seqs"], per, dtype=torch.int32, device=dev)
    held = torch.from_numpy(np.arange(per)[None, :] < need[:, None]).to(dev)
    table[held] = order[:int(need.sum())]
    starts = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).to(dev)
    return dict(pool=pool, table=table, starts=starts, lens=torch.from_numpy(lens.astype(np.int32)).to(dev), pages=pages, rows=int(new.sum()))


def prepare(case, seed):
    if own:      # the calls run on their context's stream: a program that mixes them with torch's work makes it torch's stream too, once
        torch.cuda.set_stream(_framework().stream)
    c, dev = case, torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 1000003 + 17)
    s = dict(c=c)
    kind = c["kind"]
    if kind == "rotate":
        # a joint projection's rows: the heads that turn, then as many columns that do not
        s["x"] = torch.randn(c["tokens"], c["heads"] * c["dim"] + 512, generator=g, device=dev).to(FLOATS[c["type"]])
        first = torch.randint(0, 100000, (c["axes"], 1), generator=g, device=dev)
        step = torch.tensor([[1], [7], [3]], device=dev)[:c["axes"]]
        s["positions"] = (first + torch.arange(c["tokens"], device=dev)[None, :] * step % 20011).to(torch.int32)
        return s
    if kind == "verify":
        b, k, v = c["seqs"], c["drafts"], c["vocab"]
        logits = 3 * torch.randn(b, k + 1, v, generator=g, device=dev)
        other = c["near"] * logits[:, :k] + math.sqrt(1 - c["near"] ** 2) * 3 * torch.randn(b, k, v, generator=g, device=dev)
        s["target"] = torch.softmax(logits, -1)
        s["draft"] = torch.softmax(other, -1)
        s["tokens"] = torch.multinomial(s["draft"].view(b * k, v), 1, generator=g).view(b, k).to(torch.int32)
        if not c["sampled"]:
            s["draft"] = None
        s["counts"] = torch.from_numpy((k - (np.arange(b) * 5) % (k + 1)).astype(np.int32)).to(dev) if c["ragged"] else None
        s["uniform"] = torch.rand(b, k + 1, generator=g, device=dev)
        return s
    s.update(_pool(c, g, dev))
    t = FLOATS[c["type"]]
    if kind == "attend":
        s["q"] = (1.5 * torch.randn(s["rows"], c["heads"] * c["dim"], generator=g, device=dev)).to(t)
        s["sinks"] = torch.randn(c["heads"], generator=g, device=dev) if c["sinks"] else None
    elif kind == "store":
        # rows of a joint projection; a few channels are far larger than the rest, as in trained models
        wide = c["kv_heads"] * c["dim"]
        x = torch.randn(s["rows"], 2 * wide, generator=g, device=dev)
        x[:, ::61] *= 8
        s["kv"] = x.to(t)
    return s


# ---- the plain form --------------------------------------------------------------------------------------------------------------

def _values(c, codes, scales):
    """what stored rows stand for, in 32 bits"""
    if c["cache"] in ("f16", "bf16"):
        return codes.float()
    if c["cache"] == "q4_0":
        b = codes.unflatten(-1, (-1, 16))
        codes = torch.cat([b & 15, b >> 4], -1).flatten(-2).float() - 8
    return (codes.float().unflatten(-1, (-1, 32)) * scales.float()[..., None]).flatten(-2)


def _quantise(c, x):
    """rows of 32-bit numbers as they are stored: (codes, scales)"""
    if c["cache"] in ("f16", "bf16"):
        return x.to(torch.float16 if c["cache"] == "f16" else torch.bfloat16), None
    b = x.unflatten(-1, (-1, 32))
    hi, lo = b.amax(-1), b.amin(-1)
    if c["cache"] == "q8_0":
        d = (torch.maximum(hi, -lo) * torch.tensor(1 / 127, dtype=torch.float32, device=x.device)).clamp(max=515.5).half()
    else:
        d = (torch.where(hi >= -lo, hi, lo) * -0.125).clamp(-8188, 8188).half()
    inv = torch.where(d == 0, torch.zeros((), device=x.device), torch.ones_like(hi) / d.float())
    code = torch.round(b * inv[..., None])
    if c["cache"] == "q8_0":
        return code.clamp(-127, 127).to(torch.int8).flatten(-2), d
    code = code.clamp(-8, 7).to(torch.int32) + 8
    return (code[..., :16] | code[..., 16:] << 4).to(torch.uint8).flatten(-2), d


def _places(s):
    """of each new row its sequence, position, page and place in the page"""
    row = torch.arange(s["rows"], device=s["pool"].device)
    seq = torch.searchsorted(s["starts"][1:].long(), row, right=True)
    pos = s["lens"].long()[seq] - (s["starts"].long()[seq + 1] - row)
    return seq, pos, s["table"][seq, pos // s["c"]["page"]].long(), pos % s["c"]["page"]


def _read(s):
    c = s["c"]
    _, _, page, at = _places(s)
    return [_values(c, codes[page, :, at], None if scales is None else scales[page, :, at]).to(FLOATS[c["type"]]) for codes, scales in _parts(c, s["pool"])]


def _store(s):
    c = s["c"]
    _, _, page, at = _places(s)
    rows = s["kv"].float().view(s["rows"], 2, c["kv_heads"], c["dim"])
    (kc, ks), (vc, vs) = _parts(c, s["pool"])
    (kq, kd), (vq, vd) = _quantise(c, rows[:, 0]), _quantise(c, rows[:, 1])
    kc[page, :, at] = kq
    vc[page, :, at] = vq
    if ks is not None:
        ks[page, :, at] = kd
        vs[page, :, at] = vd
    return _read(s)


def _attend(s):
    c, dev = s["c"], s["pool"].device
    group, kvh, dim, b = c["heads"] // c["kv_heads"], c["kv_heads"], c["dim"], c["seqs"]
    seq, pos, _, _ = _places(s)
    new, most = (s["starts"][1:] - s["starts"][:-1]).long(), int(_lengths(c)[1].max())
    q = torch.zeros(b, most, c["heads"], dim, device=dev)
    row = torch.arange(s["rows"], device=dev) - s["starts"].long()[seq]
    q[seq, row] = s["q"].float().view(-1, c["heads"], dim)
    q = q.view(b, most, kvh, group, dim).permute(0, 2, 1, 3, 4).reshape(b, kvh, most * group, dim)
    k, v = (_values(c, codes[s["table"].long()], None if scales is None else scales[s["table"].long()]).transpose(1, 2).flatten(2, 3) for codes, scales in _parts(c, s["pool"]))
    at = (s["lens"].long() - new)[:, None] + torch.arange(most, device=dev)      # position of each row
    key = torch.arange(k.shape[2], device=dev)
    seen = (key <= at[..., None]) & (at[..., None] < s["lens"].long()[:, None, None])
    if c["window"]:
        seen &= key > at[..., None] - c["window"]
    score = torch.matmul(q, k.transpose(-1, -2)) * (1 / math.sqrt(dim))
    score = score.view(b, kvh, most, group, -1).masked_fill_(~seen[:, None, :, None], -math.inf).view(b, kvh, most * group, -1)
    top = score.amax(-1, keepdim=True)
    if c["sinks"]:
        sink = s["sinks"].view(1, kvh, 1, group).expand(b, kvh, most, group).reshape(b, kvh, most * group, 1)
        top = torch.maximum(top, sink)
    top = top.clamp(min=-1e30)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    if c["sinks"]:
        total = total + torch.exp(sink - top)
    out = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.view(b, kvh, most, group, dim).permute(0, 2, 1, 3, 4).reshape(b, most, c["heads"] * dim)
    return out[seq, row].to(FLOATS[c["type"]])


def _sections(c):
    """pairs of a head that each axis turns"""
    half = c["rot"] // 2
    return {1: (half, 0, 0), 2: (half // 2, half - half // 2, 0), 3: (half // 4, (half - half // 4) // 2, half - half // 4 - (half - half // 4) // 2)}[c["axes"]]


def _rotate(s):
    c, dev = s["c"], s["x"].device
    half, heads, dim = c["rot"] // 2, c["heads"], c["dim"]
    axis = torch.repeat_interleave(torch.arange(3, device=dev), torch.tensor(_sections(c), device=dev))
    angle = s["positions"].double()[axis].T * torch.exp(torch.arange(half, device=dev, dtype=torch.float64) * (-2 / c["rot"] * math.log(c["base"])))
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    x = s["x"][:, :heads * dim].float().view(-1, heads, dim)
    t = x[..., :c["rot"]]
    a, b = (t[..., :half], t[..., half:]) if c["pairs"] == "halves" else (t[..., 0::2], t[..., 1::2])
    a, b = a * cos - b * sin, a * sin + b * cos
    t = torch.cat([a, b], -1) if c["pairs"] == "halves" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([t, x[..., c["rot"]:]], -1).to(s["x"].dtype).view(-1, heads * dim)


def _verify(s):
    c, dev = s["c"], s["target"].device
    b, k = c["seqs"], c["drafts"]
    i, each = torch.arange(k, device=dev), torch.arange(b, device=dev)
    x = s["tokens"].long()
    counts = s["counts"].long() if s["counts"] is not None else torch.full((b,), k, device=dev)
    p = s["target"][:, :k].gather(2, x[..., None])[..., 0].double()
    q = s["draft"].gather(2, x[..., None])[..., 0].double() if s["draft"] is not None else torch.ones_like(p)
    stands = (s["uniform"][:, :k].double() * q < p) & (i < counts[:, None])
    accepted = stands.long().cumprod(1).sum(1)
    refused = accepted < counts
    w = s["target"][each, accepted].double()
    at = accepted.clamp(max=k - 1)
    if s["draft"] is not None:
        less = s["draft"][each, at].double()
    else:
        less = torch.zeros_like(w).scatter_(1, x.gather(1, at[:, None]), math.inf)
    rest = (w - torch.where(refused[:, None], less, torch.zeros_like(less))).clamp(min=0)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, w)
    running = rest.cumsum(1)
    drawn = (running <= s["uniform"][:, k:].double() * running[:, -1:]).sum(1).clamp(max=c["vocab"] - 1)
    j = torch.arange(k + 1, device=dev)
    tokens = torch.where(j < accepted[:, None], torch.cat([x, x[:, :1]], 1), torch.full_like(x[:, :1], -1))
    tokens = torch.where(j == accepted[:, None], drawn[:, None], tokens)
    return tokens.to(torch.int32), accepted.to(torch.int32)


# ---- the framework's calls -------------------------------------------------------------------------------------------------------

_kept = {}


class _Framework:
    """the package, a context of it on a device, the context's stream as torch knows it, and a workspace that grows"""

    def __init__(self, device):
        self.lva = importlib.import_module("llama-vulkan_amd")
        self.ctx = self.lva.Context(device)
        self.stream = torch.cuda.ExternalStream(self.ctx.stream(), device=device)
        self.stream_id = self.stream.stream_id
        self.work = torch.empty(0, dtype=torch.uint8, device=torch.device("cuda", device))

    def workspace(self, size):
        if self.work.numel() < size:
            self.ctx.sync()
            self.work = torch.empty(size, dtype=torch.uint8, device=self.work.device)
        return self.work.data_ptr()


def _framework():
    """the current device's"""
    device = torch.cuda.current_device()
    if device not in _kept:
        _kept[device] = _Framework(device)
    return _kept[device]


def _type(lva, name):
    return {"f32": lva.LV_F32, "f16": lva.LV_F16, "bf16": lva.LV_BF16, "q8_0": lva.LV_Q8_0, "q4_0": lva.LV_Q4_0}[name]


def _own(s):
    """The calls, in order with the current stream's work: as they are where the program has made the context's stream the current one, by events where it has not."""
    f = _framework()
    if torch.accelerator.current_stream().stream_id == f.stream_id:
        return _calls(f, s)
    here = torch.cuda.current_stream()
    f.stream.wait_stream(here)
    with torch.cuda.stream(f.stream):
        out = _calls(f, s)
    here.wait_stream(f.stream)
    for x in (out,) if isinstance(out, torch.Tensor) else out:
        x.record_stream(here)
    return out


def _calls(f, s):
    lva, ctx = f.lva, f.ctx
    c, dev = s["c"], torch.device("cuda", torch.cuda.current_device())
    if c["kind"] == "rotate":
        x, width = s["x"], c["heads"] * c["dim"]
        out = torch.empty(c["tokens"], width, dtype=x.dtype, device=dev)
        spec = lva.RotateSpec(c["rot"], c["base"], _sections(c), PAIRS[c["pairs"]])
        ctx.rotate(out.data_ptr(), width, x.data_ptr(), x.stride(0), _type(lva, c["type"]), s["positions"].data_ptr(), c["tokens"], c["heads"], c["dim"], spec)
        return out
    if c["kind"] == "verify":
        b, k = c["seqs"], c["drafts"]
        tokens, accepted = torch.empty(b, k + 1, dtype=torch.int32, device=dev), torch.empty(b, dtype=torch.int32, device=dev)
        batch = lva.DraftBatch(b, k, c["vocab"], s["target"].data_ptr(), c["vocab"], s["draft"].data_ptr() if s["draft"] is not None else None, c["vocab"],
                               s["tokens"].data_ptr(), s["counts"].data_ptr() if s["counts"] is not None else None, s["uniform"].data_ptr())
        size = ctx.verify_drafts_workspace(batch)
        ctx.verify_drafts(tokens.data_ptr(), accepted.data_ptr(), batch, f.workspace(size), size)
        return tokens, accepted
    cache = lva.PagedCache(s["pool"].data_ptr(), _type(lva, c["cache"]), c["kv_heads"], c["dim"], c["page"], s["pages"])
    batch = lva.PagedBatch(c["seqs"], s["rows"], s["starts"].data_ptr(), s["lens"].data_ptr(), s["table"].data_ptr(), s["table"].shape[1])
    t = _type(lva, c["type"])
    if c["kind"] == "attend":
        out = torch.empty_like(s["q"])
        spec = lva.PagedAttnSpec(c["heads"], 1 / math.sqrt(c["dim"]), c["window"], 0, s["sinks"].data_ptr() if c["sinks"] else None)
        size = ctx.paged_attention_workspace(t, cache, batch, spec)
        ctx.paged_attention(out.data_ptr(), out.stride(0), s["q"].data_ptr(), s["q"].stride(0), t, cache, batch, spec, f.workspace(size), size)
        return out
    width = c["kv_heads"] * c["dim"]
    if c["kind"] == "store":
        kv = s["kv"]
        ctx.paged_write(cache, batch, kv.data_ptr(), kv.stride(0), kv.data_ptr() + width * kv.element_size(), kv.stride(0), t)
    k, v = (torch.empty(s["rows"], c["kv_heads"], c["dim"], dtype=FLOATS[c["type"]], device=dev) for _ in range(2))
    ctx.paged_read(cache, batch, k.data_ptr(), width, v.data_ptr(), width, t)
    return [k, v]


def run(state):
    if own:
        return _own(state)
    return {"rotate": _rotate, "verify": _verify, "attend": _attend, "store": _store, "load": _read}[state["c"]["kind"]](state)


# ---- in 64 bits, by the definitions --------------------------------------------------------------------------------------------

def _stored64(c, pool, page, at, which):
    """one sequence's rows [token][kv head][dim] of the keys (0) or the values (1), read byte by byte's meaning from the layout"""
    cb, sb = _row_bytes(c)
    base = which * c["page"] * (cb + sb)
    n, heads = page.numel(), c["kv_heads"]
    block = pool[page]                                              # [n][heads][bytes]
    index = (base + at * cb)[:, None, None] + torch.arange(cb, device=pool.device)
    raw = torch.gather(block, 2, index.expand(n, heads, cb))
    if c["cache"] in ("f16", "bf16"):
        return raw.view(FLOATS[c["cache"]]).double()
    index = (base + c["page"] * cb + at * sb)[:, None, None] + torch.arange(sb, device=pool.device)
    d = torch.gather(block, 2, index.expand(n, heads, sb)).view(torch.float16).double().repeat_interleave(32, -1)
    if c["cache"] == "q8_0":
        return raw.view(torch.int8).double() * d
    raw = raw.view(n, heads, -1, 16).long()
    return (torch.stack([raw % 16, raw // 16], 3).reshape(n, heads, -1).double() - 8) * d


def _sequence64(s, b, lo, hi):
    """keys and values of positions lo .. hi - 1 of a sequence"""
    p = torch.arange(lo, hi, device=s["pool"].device)
    page = s["table"][b].long()[p // s["c"]["page"]]
    return [_stored64(s["c"], s["pool"], page, p % s["c"]["page"], which) for which in (0, 1)]


def _exact_store(c, x):
    """the number nearest to each of 64-bit x that its block's scale can express"""
    if c["cache"] in ("f16", "bf16"):
        return x.to(FLOATS[c["cache"]]).double()
    b = x.reshape(*x.shape[:-1], -1, 32)
    big = b.abs().amax(-1, keepdim=True)
    if c["cache"] == "q8_0":
        d = (big / 127).clamp(max=515.5)
        lo, hi = -127, 127
    else:
        signed = torch.where(b.amax(-1, keepdim=True) >= big, big, -big)
        d = (signed / -8).clamp(-8188, 8188)
        lo, hi = -8, 7
    d = d.float().half().double()
    return (torch.where(d != 0, torch.round(b / torch.where(d != 0, d, torch.ones_like(d))), torch.zeros_like(b)).clamp(lo, hi) * d).reshape(x.shape)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    kind = c["kind"]
    if kind == "verify":
        return None                                                 # whole numbers
    if kind == "rotate":
        x = s["x"][:, :c["heads"] * c["dim"]].double().view(c["tokens"], c["heads"], c["dim"]).clone()
        pair = 0
        for axis, pairs in enumerate(_sections(c)):
            for _ in range(pairs):
                a, b = (pair, pair + c["rot"] // 2) if c["pairs"] == "halves" else (2 * pair, 2 * pair + 1)
                turn = s["positions"][axis].double() * c["base"] ** (-2 * pair / c["rot"])
                z = torch.complex(x[..., a], x[..., b]) * torch.polar(torch.ones_like(turn), turn)[:, None]
                x[..., a], x[..., b] = z.real, z.imag
                pair += 1
        return x.view(c["tokens"], -1)
    lens, new = _lengths(c)
    if kind == "store":
        rows = s["kv"].double().view(s["rows"], 2, c["kv_heads"], c["dim"])
        return [_exact_store(c, rows[:, 0]), _exact_store(c, rows[:, 1])]
    if kind == "load":
        per = [_sequence64(s, b, 0, int(lens[b])) for b in range(c["seqs"])]
        return [torch.cat([p[which] for p in per]) for which in (0, 1)]
    out = torch.zeros(s["rows"], c["heads"], c["dim"], dtype=torch.float64, device=s["pool"].device)
    group, row0 = c["heads"] // c["kv_heads"], 0
    for b in range(c["seqs"]):
        n, m = int(lens[b]), int(new[b])
        lo = max(0, n - m + 1 - c["window"]) if c["window"] else 0
        k, v = _sequence64(s, b, lo, n)
        pos = torch.arange(n - m, n, device=k.device)[:, None]
        key = torch.arange(lo, n, device=k.device)[None, :]
        hidden = (key > pos) | ((key <= pos - c["window"]) if c["window"] else torch.zeros_like(key > pos))
        for h in range(c["heads"]):
            q = s["q"][row0:row0 + m, h * c["dim"]:(h + 1) * c["dim"]].double()
            score = (q @ k[:, h // group].T) / math.sqrt(c["dim"])
            score = score.masked_fill(hidden, -math.inf)
            if c["sinks"]:
                score = torch.cat([score, s["sinks"][h].double().expand(m, 1)], 1)
            p = torch.softmax(score, 1)
            out[row0:row0 + m, h] = p[:, :n - lo] @ v[:, h // group]
        row0 += m
    return out.view(s["rows"], -1)
