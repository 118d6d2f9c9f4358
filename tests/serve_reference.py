"""The operators of a serving step in double precision, straight from their definitions, and a paged cache built byte by byte from its described
layout.  Shares nothing with the product."""
import numpy as np

F32, F16, Q4, Q8, BF16 = 0, 1, 2, 8, 30
NAMES = {F32: "f32", F16: "f16", Q4: "q4_0", Q8: "q8_0", BF16: "bf16"}
BYTES = {F32: 4, F16: 2, BF16: 2}
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}      # of a rounding, relative to the value
NO_PAGE = 0xFFFFFFFF


# ---- number types ------------------------------------------------------------------------------------------------------------
def to_bf16(x):
    """bits of the nearest bf16, ties to even; NaN stays NaN"""
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    nan = (u & 0x7FFFFFFF) > 0x7F800000
    r[nan] = 0x7FC0
    return r


def from_bf16(b):
    return (np.asarray(b, dtype=np.uint16).astype(np.uint32) << 16).view(np.float32)


def encode(x, kind):
    """an array as its memory holds it"""
    with np.errstate(over="ignore"):
        x = np.asarray(x, dtype=np.float32)
        return x if kind == F32 else x.astype(np.float16) if kind == F16 else to_bf16(x)


def decode(x, kind):
    return x.astype(np.float64) if kind in (F32, F16) else from_bf16(x).astype(np.float64)


DTYPE = {F32: np.float32, F16: np.float16, BF16: np.uint16}


# ---- stored rows ---------------------------------------------------------------------------------------------------------------
def quantise(x, kind):
    """codes (int) and fp16 scales of blocks of 32 along the last axis, step by step in fp32"""
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        b = np.asarray(x, dtype=np.float32).reshape(*x.shape[:-1], -1, 32)
        clean = np.where(np.isnan(b), np.float32(0), b)
        some = ~np.isnan(b).all(-1)
        hi = np.where(some, np.where(np.isnan(b), -np.inf, b).max(-1), 0).astype(np.float32)
        lo = np.where(some, np.where(np.isnan(b), np.inf, b).min(-1), 0).astype(np.float32)
        if kind == Q8:
            d = np.minimum(np.maximum(hi, -lo) * np.float32(1.0 / 127.0), np.float32(515.5))
            low, high = -127, 127
        else:
            d = np.clip(np.where(hi >= -lo, hi, lo) * np.float32(-0.125), np.float32(-8188), np.float32(8188))
            low, high = -8, 7
        d = d.astype(np.float16)
        d[d == 0] = 0                                   # not -0
        f = d.astype(np.float32)
        inv = np.where(f == 0, np.float32(0), np.float32(1) / f).astype(np.float32)
        code = np.clip(np.rint((clean * inv[..., None]).astype(np.float32)), low, high)
        code = np.where(np.isnan(b) | (inv == 0)[..., None], 0, code)
    return code.astype(np.int32), d


def stored_values(x, kind):
    """what rows of numbers become when they are stored, in double"""
    if kind in (F16, BF16):
        return decode(encode(x, kind), kind)
    code, d = quantise(x, kind)
    return (code * d.astype(np.float64)[..., None]).reshape(x.shape)


class Pool:
    """a paged cache on the host: bytes [pages][kv heads][block]"""

    def __init__(self, kind, kv_heads, dim, page, pages, rng=None):
        self.kind, self.kv_heads, self.dim, self.page, self.pages = kind, kv_heads, dim, page, pages
        self.code_row = {F16: 2 * dim, BF16: 2 * dim, Q8: dim, Q4: dim // 2}[kind]
        self.scale_row = dim // 16 if kind in (Q8, Q4) else 0
        self.half = page * (self.code_row + self.scale_row)
        self.block = 2 * self.half
        self.bytes = np.zeros((pages, kv_heads, self.block), dtype=np.uint8)
        if rng is not None:      # what earlier users of the pages left: anything, not finite numbers among it
            self.bytes[:] = rng.integers(0, 256, self.bytes.shape, dtype=np.uint8)

    def row(self, page, head, which, at):
        """(codes, scales) of one row as byte slices"""
        b = self.bytes[page, head, which * self.half:(which + 1) * self.half]
        s = self.page * self.code_row
        return b[at * self.code_row:(at + 1) * self.code_row], b[s + at * self.scale_row:s + (at + 1) * self.scale_row]

    def put(self, page, head, which, at, x):
        codes, scales = self.row(page, head, which, at)
        if self.kind in (F16, BF16):
            codes[:] = encode(x, self.kind).view(np.uint8)
            return
        q, d = quantise(np.asarray(x, dtype=np.float32), self.kind)
        scales[:] = d.view(np.uint8)
        if self.kind == Q8:
            codes[:] = q.astype(np.int8).reshape(-1).view(np.uint8)
        else:
            q = (q + 8).astype(np.uint8)
            codes[:] = (q[:, :16] | (q[:, 16:] << 4)).reshape(-1)

    def get(self, page, head, which, at):
        codes, scales = self.row(page, head, which, at)
        if self.kind == F16:
            return codes.view(np.float16).astype(np.float64)
        if self.kind == BF16:
            return from_bf16(codes.view(np.uint16)).astype(np.float64)
        d = scales.view(np.float16).astype(np.float64)[:, None]
        if self.kind == Q8:
            return (codes.view(np.int8).astype(np.float64).reshape(-1, 32) * d).reshape(-1)
        b = codes.reshape(-1, 16)
        return ((np.concatenate([b & 15, b >> 4], 1).astype(np.float64) - 8) * d).reshape(-1)


class Step:
    """lens and new tokens of sequences, with pages of a pool in random order; pad: rows behind the last sequence's"""

    def __init__(self, pool, lens, new, rng, extra_columns=1, pad=0):
        self.lens, self.new, self.pad = np.asarray(lens, dtype=np.int64), np.asarray(new, dtype=np.int64), pad
        need = -(-self.lens // pool.page)
        self.table = np.full((len(lens), int(need.max(initial=0)) + extra_columns), NO_PAGE, dtype=np.uint32)
        order = rng.permutation(pool.pages)[:int(need.sum())]
        assert len(order) == need.sum(), "the pool is too small"
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.starts = np.concatenate([[0], np.cumsum(self.new)]).astype(np.uint32)
        self.tokens = int(self.starts[-1]) + pad

    def place(self, pool, b, position):
        """(page, place) of a position, or None"""
        i = position // pool.page
        if position < 0 or i >= self.table.shape[1] or self.table[b, i] >= pool.pages:
            return None
        return int(self.table[b, i]), position % pool.page

    def rows(self):
        """(row, sequence, position) of every new token"""
        for b in range(len(self.lens)):
            for i in range(int(self.new[b])):
                yield int(self.starts[b]) + i, b, int(self.lens[b] - self.new[b]) + i


# ---- attention -----------------------------------------------------------------------------------------------------------------
def attention(pool, step, q, heads, scale, window=0, chunk=0, sinks=None):
    """q [tokens][heads][dim] in double.  Returns out, sum of p |v| (what relative errors of weights and values are relative to), and the largest scale * sum |q| |k| of
    a row's keys (what rounding errors of its scores are relative to), the keys seen, and the sum of their |v|"""
    group = heads // pool.kv_heads
    out, size, mass = np.zeros_like(q), np.zeros_like(q), np.zeros_like(q)
    reach, seen = np.zeros(q.shape[:2]), np.zeros(q.shape[0], dtype=np.int64)
    cache = {}
    with np.errstate(invalid="ignore", over="ignore"):
        for row, b, pos in step.rows():
            lo = 0
            if window:
                lo = max(lo, pos - window + 1)
            if chunk and pos >= 0:
                lo = max(lo, pos - pos % chunk)
            keys = [p for p in range(lo, pos + 1) if step.place(pool, b, p) is not None]
            seen[row] = len(keys)
            if not keys:
                continue
            for kvh in range(pool.kv_heads):
                k, v = [], []
                for p in keys:
                    if (b, p, kvh) not in cache:
                        page, at = step.place(pool, b, p)
                        cache[b, p, kvh] = pool.get(page, kvh, 0, at), pool.get(page, kvh, 1, at)
                    k.append(cache[b, p, kvh][0])
                    v.append(cache[b, p, kvh][1])
                k, v = np.array(k), np.array(v)
                for h in range(kvh * group, (kvh + 1) * group):
                    s = scale * (k @ q[row, h])
                    top = max(s.max(), sinks[h]) if sinks is not None else s.max()
                    p = np.exp(s - top)
                    total = p.sum() + (np.exp(sinks[h] - top) if sinks is not None else 0)
                    out[row, h] = (p[:, None] * v).sum(0) / total
                    size[row, h] = (p[:, None] * np.abs(v)).sum(0) / total
                    mass[row, h] = np.abs(v).sum(0)
                    reach[row, h] = np.max(np.abs(scale) * (np.abs(k) @ np.abs(q[row, h])))
    return out, size, reach, seen, mass


def attention_bound(want, size, reach, seen, mass, dim, kind, cache):
    """How far a kernel's result may be off.  Scores: products of exact operands (32-bit queries as pieces of 22 bits or more) summed in fp32, dim + 8 roundings of at most
    2^-24 of sum |q k|, 2^-22 for the pieces; an error e of a score is one of e (and e of the maximum) in a weight's exponent.  Weights: exp2 to 2^-22, the sum over `seen` keys in
    fp32, and rounded to the matrix cores' operands: fp16 2^-11, bf16 2^-8 where the result is bf16 too (two pieces of it 2^-16), two pieces of fp16 2^-22.  Values of blocks are scaled in fp16 (2^-11) where the result is
    16-bit.  The sums over keys are fp32 (`seen` roundings at most), then the result is rounded once.
    Numbers next to 0: weights enter fp16 products in units where a row's largest one (of the keys so far) is 2^12, in the kernel for chunks, whose results are 16-bit, 2^6 to 2^14.
    Below 2^-14 a rounding is one of 2^-25 whatever the number, so each weight may be off by 2^-37 or 2^-31 of the largest, which is no more than the sum: so much times sum |v| of the
    result.  Scaled 16-bit values: 2^-25 times weights of sum 1."""
    blocks = cache in (Q8, Q4)
    if kind == F32:
        weight, value = 2.0 ** -21, 0.0
    elif cache == BF16:
        weight, value = 2.0 ** -8 if kind == BF16 else 2.0 ** -16, 0.0
    else:
        weight, value = 2.0 ** -11, 2.0 ** -11 if blocks else 0.0
    score = reach[..., None] * ((dim + 8) * 2.0 ** -24 + 2.0 ** -22)
    relative = 2 * score + 2.0 ** -20 + 2 * (seen[:, None, None] + 64) * 2.0 ** -24 + weight + value
    small = (0 if cache == BF16 else (2.0 ** -37 if kind == F32 else 2.0 ** -31) * mass) + (2.0 ** -25 if value else 0)
    return HALF_STEP[kind] * np.abs(want) * 1.01 + relative * (1 + relative) * 1.1 * size + small + (2.0 ** -24 if kind == F16 else 1e-37)


# ---- rotation ------------------------------------------------------------------------------------------------------------------
def rotate(x, positions, rot, base, sections=(0, 0, 0), halves=False, per_axis=False):
    """x [tokens][heads][dim], positions [axes][tokens]; returns the turned rows and |a| + |b| of each element's pair"""
    x = np.array(x, dtype=np.float64)
    size = np.zeros_like(x)
    sections = tuple(sections) if sum(sections) else (rot // 2, 0, 0)
    pair = 0
    for axis, n in enumerate(sections):
        for i in range(n):
            a, b = (pair, pair + rot // 2) if halves else (2 * pair, 2 * pair + 1)
            angle = positions[axis].astype(np.float64) * base ** (-(i / n) if per_axis else -2.0 * pair / rot)
            z = (x[..., a] + 1j * x[..., b]) * np.exp(1j * angle)[:, None]
            size[..., a] = size[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
            x[..., a], x[..., b] = z.real, z.imag
            pair += 1
    return x, size


# ---- verification --------------------------------------------------------------------------------------------------------------
def verify(target, draft, tokens, counts, uniforms):
    """target [seqs][drafts + 1][vocab], draft the same without the last row or None -> tokens [seqs][drafts + 1], accepted [seqs]"""
    seqs, drafts = tokens.shape
    vocab = target.shape[2]
    out, accepted = np.full((seqs, drafts + 1), 0xFFFFFFFF, dtype=np.uint32), np.zeros(seqs, dtype=np.uint32)
    with np.errstate(invalid="ignore"):
        for b in range(seqs):
            n, r = min(int(counts[b]), drafts), 0
            while r < n:
                x = int(tokens[b, r])
                q = 1.0 if draft is None else float(draft[b, r, x]) if x < vocab else 0.0
                if x >= vocab or not float(uniforms[b, r]) * q < float(target[b, r, x]):
                    break
                out[b, r] = x
                r += 1
            p = target[b, r].astype(np.float64)
            w = p.copy()
            if r < n:
                if draft is not None:
                    w = p - draft[b, r].astype(np.float64)
                elif tokens[b, r] < vocab:
                    w[int(tokens[b, r])] = 0
            w = np.where(w > 0, w, 0)
            if not w.sum() > 0:
                w = np.where(p > 0, p, 0)
            pick = 0
            if w.sum() > 0:
                over = np.cumsum(w) > float(uniforms[b, drafts]) * w.sum()
                pick = int(np.argmax(over)) if over.any() else int(np.nonzero(w)[0][-1])
            out[b, r] = pick
            accepted[b] = r
    return out, accepted
