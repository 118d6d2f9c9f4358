"""A serving step's operators on the GPU against their definitions in double precision (tests/serve_reference.py), through the C-ABI."""
import ctypes as C

import numpy as np
import pytest

import serve_reference as ref
from serve_reference import BF16, F16, F32, HALF_STEP, NO_PAGE, Q4, Q8

pytestmark = pytest.mark.gpu

KINDS = dict(ids=lambda k: ref.NAMES[k])


class Device:
    """device arrays of a test, freed at its end"""

    def __init__(self, lva, ctx):
        self.lva, self.ctx, self.held = lva, ctx, []

    def put(self, a):
        a = np.ascontiguousarray(a)
        p = self.ctx.to_device(a if a.size else np.zeros(4, np.uint8))
        self.held.append(p)
        return p

    def get(self, p, shape, dtype):
        return self.ctx.to_host(p, shape, dtype)

    def cache(self, pool):
        p = self.put(pool.bytes)
        return p, self.lva.PagedCache(p.value, pool.kind, pool.kv_heads, pool.dim, pool.page, pool.pages)

    def batch(self, step):
        return self.lva.PagedBatch(len(step.lens), step.tokens, self.put(step.starts).value, self.put(step.lens.astype(np.uint32)).value, self.put(step.table).value,
                                   step.table.shape[1])


@pytest.fixture
def dev(lva, ctx):
    d = Device(lva, ctx)
    yield d
    ctx.sync()
    for p in d.held:
        ctx.free(p)


def strided(x, kind, extra):
    """rows with `extra` elements behind each that nobody may touch: (array as memory, stride)"""
    rows = x.reshape(x.shape[0], -1)
    out = ref.encode(np.full((rows.shape[0], rows.shape[1] + extra), 3.25), kind)
    out[:, :rows.shape[1]] = ref.encode(rows, kind)
    return out, rows.shape[1] + extra


# ---- rotation ----------------------------------------------------------------------------------------------------------------
ROTATIONS = [
    # tokens, heads, dim, rot, base, sections, halves, per axis
    (1, 1, 8, 8, 1e4, (0, 0, 0), False, False),
    (1, 64, 128, 128, 1e4, (0, 0, 0), False, False),
    (7, 40, 128, 128, 1e6, (16, 24, 24), True, False),
    (33, 5, 80, 80, 1e4, (8, 16, 16), True, False),          # a head size that is no power of two
    (5, 3, 64, 32, 5e5, (16, 0, 0), True, False),            # half of the head stays
    (5, 3, 64, 32, 5e5, (5, 11, 0), False, False),
    (9, 2, 128, 40, 1e4, (0, 0, 0), True, False),            # pairs one by one: 20 is no multiple of 8
    (9, 2, 128, 42, 1e4, (7, 7, 7), False, False),
    (4, 7, 72, 72, 1e4, (12, 12, 12), False, True),          # every axis its own frequencies
    (4, 7, 96, 96, 1e4, (0, 24, 24), True, True),            # a first axis that turns nothing
    (3, 2, 512, 512, 1e4, (0, 0, 0), True, False),
    (3, 2, 24, 0, 1e4, (0, 0, 0), False, False),             # nothing turns
    (3000, 3, 32, 32, 1e4, (0, 0, 0), False, False),         # more tokens than workgroups share
]


@pytest.mark.parametrize("kind", [F32, F16, BF16], **KINDS)
@pytest.mark.parametrize("shape", ROTATIONS, ids=str)
def test_rotate(lva, ctx, dev, kind, shape):
    tokens, heads, dim, rot, base, sections, halves, per_axis = shape
    rng = np.random.default_rng(11)
    x = rng.standard_normal((tokens, heads, dim)) * 2
    axes = max([i + 1 for i in range(3) if sections[i]], default=1)
    positions = rng.integers(0, 1 << 20, (axes, tokens)).astype(np.uint32)
    positions[:, 0] = (0, 1, 0xFFFFFFFF)[:axes] if tokens > 1 else 131071
    mem, ldx = strided(x, kind, 16)
    want, size = ref.rotate(ref.decode(mem[:, :heads * dim], kind).reshape(x.shape), positions, rot, base, sections, halves, per_axis)
    # angle: rounded to fp32 in half turns (pi 2^-24), double before it (2^32 turns: 2^-18 of nothing); sine, cosine, products and sum: 4 roundings
    bound = (np.pi * 2.0 ** -24 + 2.0 ** -20 + 4 * 2.0 ** -24) * size + HALF_STEP[kind] * np.abs(want) + (2.0 ** -24 if kind == F16 else 0)
    spec = lva.RotateSpec(rot, base, sections, (lva.ROTATE_HALVES if halves else 0) | (lva.ROTATE_PER_AXIS if per_axis else 0))
    dx, dp = dev.put(mem), dev.put(positions)
    out0 = np.zeros((tokens + 1, heads * dim + 32), dtype=mem.dtype)
    out0[:] = ref.encode(np.full(out0.shape, -7.5), kind)
    dout = dev.put(out0)
    ctx.rotate(dout, heads * dim + 32, dx, ldx, kind, dp, tokens, heads, dim, spec)
    got = dev.get(dout, out0.shape, out0.dtype)
    assert np.all(np.abs(ref.decode(got[:tokens, :heads * dim], kind).reshape(x.shape) - want) <= bound)
    assert np.array_equal(got[:, heads * dim:], out0[:, heads * dim:]) and np.array_equal(got[tokens], out0[tokens])
    # in place: the same bits
    ctx.rotate(dx, ldx, dx, ldx, kind, dp, tokens, heads, dim, spec)
    again = dev.get(dx, mem.shape, mem.dtype)
    assert np.array_equal(again[:, :heads * dim], got[:tokens, :heads * dim]) and np.array_equal(again[:, heads * dim:], mem[:, heads * dim:])


def test_rotate_nothing(lva, ctx):
    spec = lva.RotateSpec(128, 1e4, (0, 0, 0), 0)
    ctx.rotate(None, 0, None, 0, F32, None, 0, 4, 128, spec)


# ---- rows to pages and back --------------------------------------------------------------------------------------------------------
def odd_numbers(rng, shape):
    """rows as a model has them, and blocks with everything that can go wrong"""
    x = (rng.standard_normal(shape) * rng.choice([1e-6, 1e-2, 1, 50], (*shape[:-1], 1))).astype(np.float32)
    flat = x.reshape(-1, 32)
    n = len(flat)
    flat[0 % n] = 0
    flat[1 % n, :4] = (np.inf, -1, 2, 3)
    flat[2 % n, 5] = np.nan
    flat[3 % n] = np.nan
    flat[4 % n, :2] = (-np.inf, np.inf)
    flat[5 % n] = 1e-9                                   # its scale is 0 in fp16
    flat[6 % n, :2] = (4.0, -4.0)                        # of two furthest ones the positive
    flat[7 % n] = np.arange(-16, 16) * 0.5               # ties
    flat[8 % n] = (np.arange(32) - 15.5) * 127 / 15.5    # scale next to 1
    flat[9 % n, 0] = 3e38
    flat[10 % n] = 7e-6                                  # a subnormal scale
    flat[11 % n, 31] = -70000
    return x


@pytest.mark.parametrize("kind", [F32, F16, BF16], **KINDS)
@pytest.mark.parametrize("cache", [F16, BF16, Q8, Q4], **KINDS)
@pytest.mark.parametrize("kv_heads,dim,page,lens,new", [
    (1, 32, 16, [1], [1]), (2, 64, 16, [40, 17, 33], [33, 0, 17]), (3, 128, 64, [65, 128, 1, 0], [2, 64, 1, 0]), (1, 256, 32, [100], [70]), (8, 128, 128, [5] * 70, [1] * 70),
], ids=str)
def test_write_and_read(lva, ctx, dev, kind, cache, kv_heads, dim, page, lens, new):
    rng = np.random.default_rng(21)
    pool = ref.Pool(cache, kv_heads, dim, page, sum(-(-n // page) for n in lens) + 3, rng)
    step = ref.Step(pool, lens, new, rng, pad=2)
    x = odd_numbers(rng, (step.tokens, 2, kv_heads, dim))
    mem, ld = strided(x, kind, 24)
    held = ref.decode(mem[:, :2 * kv_heads * dim], kind).astype(np.float32).reshape(x.shape)      # what the rows say after their own rounding
    dpool, c = dev.cache(pool)
    b = dev.batch(step)
    rows = dev.put(mem)
    width = kv_heads * dim
    ctx.paged_write(c, b, rows, ld, rows.value + width * mem.itemsize, ld, kind)
    for row, seq, pos in step.rows():
        p, at = step.place(pool, seq, pos)
        for which in (0, 1):
            for h in range(kv_heads):
                pool.put(p, h, which, at, held[row, which, h])
    got = dev.get(dpool, pool.bytes.shape, np.uint8)
    if cache in (F16, BF16):      # a NaN's bits are its own business
        a, w = got.view(np.uint16), pool.bytes.view(np.uint16)
        exp = 0x7C00 if cache == F16 else 0x7F80
        nan = ((w & exp) == exp) & ((w & ~np.uint16(exp) & 0x7FFF) != 0)
        assert np.array_equal(a[~nan], w[~nan])
        assert np.all(((a[nan] & exp) == exp) & ((a[nan] & ~np.uint16(exp) & 0x7FFF) != 0))
    else:
        assert np.array_equal(got, pool.bytes)
    # back, with two strides
    back = ref.encode(np.full((2, step.tokens, width + 8), -7.5), kind)
    dk, dv = dev.put(back[0]), dev.put(back[1])
    ctx.paged_read(c, b, dk, width + 8, dv, width + 8, kind)
    for which, p in enumerate((dk, dv)):
        out = dev.get(p, back[0].shape, back.dtype)
        want = back[which].copy()
        for row, seq, pos in step.rows():
            place = step.place(pool, seq, pos)
            want[row, :width] = ref.encode(np.concatenate([pool.get(place[0], h, which, place[1]) for h in range(kv_heads)]), kind)
        a, w = ref.decode(out, kind), ref.decode(want, kind)
        assert np.array_equal(a, w, equal_nan=True)


def test_write_and_read_leave_what_has_no_page(lva, ctx, dev):
    """pages outside the pool, positions beyond the table and before 0, rows behind the last sequence"""
    rng = np.random.default_rng(22)
    pool = ref.Pool(Q8, 2, 64, 16, 6, rng)
    step = ref.Step(pool, [40, 20], [40, 20], rng, extra_columns=0, pad=3)
    step.table[0, 1] = 6              # the pool's end
    step.table[1, 0] = NO_PAGE
    step.table[1, 2] = 0xFFFFFFF0
    step.lens[0] = 60                 # the last 12 positions are beyond the table's 48
    step.new = np.array([40, 30])     # the second one's first 10 are before 0
    step.starts = np.array([0, 40, 70], dtype=np.uint32)
    step.tokens = 75
    x = rng.standard_normal((75, 2, 2, 64)).astype(np.float32)
    before = pool.bytes.copy()
    dpool, c = dev.cache(pool)
    b = dev.batch(step)
    rows = dev.put(x)
    ctx.paged_write(c, b, rows, 256, rows.value + 512, 256, F32)
    for row, seq, pos in step.rows():
        place = step.place(pool, seq, pos)
        if place:
            for which in (0, 1):
                for h in range(2):
                    pool.put(place[0], h, which, place[1], x[row, which, h])
    assert not np.array_equal(pool.bytes, before)
    assert np.array_equal(dev.get(dpool, pool.bytes.shape, np.uint8), pool.bytes)
    k = np.full((75, 128), -7.5, dtype=np.float32)
    dk, dv = dev.put(k), dev.put(k)
    ctx.paged_read(c, b, dk, 128, dv, 128, F32)
    want = k.copy()
    for row, seq, pos in step.rows():
        place = step.place(pool, seq, pos)
        if place:
            want[row] = np.concatenate([pool.get(place[0], h, 0, place[1]) for h in range(2)])
    assert np.array_equal(dev.get(dk, k.shape, np.float32), want)


# ---- attention ---------------------------------------------------------------------------------------------------------------------
def run_attention(dev, pool, step, q, kind, heads, scale, window=0, chunk=0, sinks=None, extra=16, fill=-7.5):
    """q [tokens][heads][dim] numbers.  Returns the result as numbers and the queries as the kernel got them; checks what lies around the result"""
    lva, ctx = dev.lva, dev.ctx
    mem, ldq = strided(q, kind, extra)
    _, c = dev.cache(pool)
    b = dev.batch(step)
    width = heads * pool.dim
    out0 = ref.encode(np.full((step.tokens + 1, width + 8), fill), kind)
    dout = dev.put(out0)
    spec = lva.PagedAttnSpec(heads, scale, window, chunk, dev.put(sinks.astype(np.float32)).value if sinks is not None else None)
    size = ctx.paged_attention_workspace(kind, c, b, spec)
    work = dev.put(np.full(size + 64, 0xFF, dtype=np.uint8))
    ctx.paged_attention(dout, width + 8, dev.put(mem), ldq, kind, c, b, spec, work if size else None, size)
    got = dev.get(dout, out0.shape, out0.dtype)
    assert np.all(dev.get(work, (size + 64,), np.uint8)[size:] == 0xFF)
    assert np.array_equal(got[:, width:], out0[:, width:])
    owned = int(step.starts[-1])
    assert np.array_equal(got[owned:], out0[owned:])
    return ref.decode(got[:owned, :width], kind).reshape(owned, heads, pool.dim), ref.decode(mem[:owned, :width], kind).reshape(owned, heads, pool.dim)


def check_attention(dev, rng, cache, kind, heads, kv_heads, dim, page, lens, new, window=0, chunk=0, sinks=False, spread=1.5, pad=0, edit=None):
    pool = ref.Pool(cache, kv_heads, dim, page, sum(-(-n // page) for n in lens) + 2, rng)
    step = ref.Step(pool, lens, new, rng, pad=pad)
    for b, n in enumerate(lens):
        for p in range(n):
            at = step.place(pool, b, p)
            for h in range(kv_heads):
                pool.put(at[0], h, 0, at[1], rng.standard_normal(dim))
                pool.put(at[0], h, 1, at[1], rng.standard_normal(dim) + 0.5)
    if edit:
        edit(pool, step)
    q = rng.standard_normal((step.tokens, heads, dim)) * spread
    s = rng.standard_normal(heads).astype(np.float32) * 2 if sinks else None
    scale = float(np.float32(dim ** -0.5))
    got, held = run_attention(dev, pool, step, q, kind, heads, scale, window, chunk, s)
    full = np.zeros((step.tokens, heads, dim))
    full[:len(held)] = held
    want, size, reach, seen, mass = (a[:len(held)] for a in ref.attention(pool, step, full, heads, scale, window, chunk, s))
    bound = ref.attention_bound(want, size, reach, seen, mass, dim, kind, cache)
    finite = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), finite)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~finite & ~np.isnan(want)], want[~finite & ~np.isnan(want)])
    off = np.abs(got[finite] - want[finite]) / bound[finite]
    assert off.size == 0 or off.max() <= 1, off.max()
    return got, want


TYPES = [(c, t) for c in (F16, BF16, Q8, Q4) for t in (F32, F16, BF16)]


@pytest.mark.parametrize("cache,kind", TYPES, ids=lambda k: ref.NAMES[k])
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_attention_of_single_tokens(dev, cache, kind, dim):
    check_attention(dev, np.random.default_rng(31), cache, kind, 4, 2, dim, 16, [1, 2, 31, 33, 130, 301], [1] * 6, pad=1)


@pytest.mark.parametrize("cache,kind", TYPES, ids=lambda k: ref.NAMES[k])
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_attention_of_chunks(dev, cache, kind, dim):
    """rows that see different keys of a tile; sequences without new tokens"""
    check_attention(dev, np.random.default_rng(32), cache, kind, 3, 1, dim, 32, [40, 50, 7, 150], [40, 0, 3, 37], pad=3)


@pytest.mark.parametrize("cache", [F16, BF16, Q8, Q4], **KINDS)
@pytest.mark.parametrize("window,chunk,sinks", [(1, 0, False), (5, 0, True), (64, 0, False), (0, 16, False), (0, 50, True), (40, 60, False), (1000, 1000, True)], ids=str)
def test_attention_masks(dev, cache, window, chunk, sinks):
    check_attention(dev, np.random.default_rng(33), cache, F16, 8, 2, 64, 16, [90, 201, 33], [70, 5, 33], window=window, chunk=chunk, sinks=sinks)
    check_attention(dev, np.random.default_rng(34), cache, F32, 2, 2, 128, 64, [90, 301], [1, 1], window=window, chunk=chunk, sinks=sinks)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 5), (12, 1), (7, 7), (32, 2)])
def test_attention_pages_and_heads(dev, page, heads, kv_heads):
    check_attention(dev, np.random.default_rng(35), Q8, BF16, heads, kv_heads, 64, page, [page - 1, page, page + 1], [1, 2, 1])


@pytest.mark.parametrize("cache,kind", TYPES, ids=lambda k: ref.NAMES[k])
def test_attention_of_one_long_sequence(dev, cache, kind):
    """cut into parts that a second launch puts together"""
    check_attention(dev, np.random.default_rng(36), cache, kind, 4, 1, 64, 64, [6001, 3], [2, 1], sinks=True)


@pytest.mark.parametrize("cache,kind", TYPES, ids=lambda k: ref.NAMES[k])
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_attention_cut_and_whole_in_one_call(dev, cache, kind, dim):
    """a table of more than 384 positions: sequences of several steps are cut, those beside them are not"""
    check_attention(dev, np.random.default_rng(50), cache, kind, 4, 2, dim, 16, [1, 130, 450, 33], [1, 1, 1, 0], pad=1, sinks=True)
    check_attention(dev, np.random.default_rng(51), cache, kind, 3, 1, dim, 32, [40, 500, 7], [40, 30, 3], pad=2)


def test_attention_of_chunks_that_are_not_cut(dev):
    """more than 384 positions and workgroups for half of the compute units: one launch, of a table that leaves nothing to cut"""
    check_attention(dev, np.random.default_rng(52), F16, F16, 32, 32, 64, 64, [700], [700])


def test_attention_of_many_sequences(dev):
    rng = np.random.default_rng(37)
    lens = rng.integers(1, 60, 150)
    check_attention(dev, rng, F16, F16, 2, 1, 64, 16, lens.tolist(), np.minimum(lens, rng.integers(0, 3, 150)).tolist())


@pytest.mark.parametrize("columns", [4, 40])
def test_attention_of_hundreds_of_sequences(dev, columns):
    """looked at 256 at a time; where the table covers more than 384 positions, the longest of them are cut"""
    rng = np.random.default_rng(59)
    lens = rng.integers(0, 40, 700)
    lens[[5, 300, 699]] = 600 if columns > 4 else 64
    new = np.minimum(lens, rng.integers(0, 3, 700))
    check_attention(dev, rng, F16, F16, 2, 1, 64, 16, lens.tolist(), new.tolist(), pad=2)


@pytest.mark.parametrize("cache,kind", [(F16, F16), (Q8, BF16), (BF16, F32)], ids=lambda k: ref.NAMES[k])
@pytest.mark.parametrize("seqs,heads,kv_heads,long,longest", [
    (100, 2, 1, (5, 70, 99), 1500),        # fewer sequences than compute units, few rows: the join has four waves a row
    (100, 12, 1, (5, 63, 64, 99), 1500),   # and one wave a row
    (150, 4, 2, (0, 64, 149), 3000),       # as many sequences' key heads as compute units: cut for evenness
    (300, 2, 2, (5, 130, 299), 5000),      # twice as many, and in longer parts
], ids=str)
def test_attention_of_more_sequences_than_a_wave_looks_at_that_are_cut(dev, cache, kind, seqs, heads, kv_heads, long, longest):
    """64 sequences are looked at at a time: what those before them take is carried on, in the launch and in the join"""
    lva, ctx = dev.lva, dev.ctx
    rng = np.random.default_rng(64)
    lens = rng.integers(1, 40, seqs)
    lens[list(long)] = [longest - 61 * i for i in range(len(long))]
    new = np.minimum(rng.integers(0, 3, seqs), lens)
    new[list(long)] = (1, 2, 1, 1)[:len(long)]
    new[1::7] = 1
    seen = {}

    def edit(pool, step):      # the call once more by itself: what has been cut is in the workspace
        seen["q"] = ref.encode(rng.standard_normal((step.tokens, heads * 64)), kind)
        _, c = dev.cache(pool)
        b, spec = dev.batch(step), lva.PagedAttnSpec(heads, 0.125, 0, 0, None)
        n = ctx.paged_attention_workspace(kind, c, b, spec)
        assert n > 0
        work, out = dev.put(np.full(n, 0xFF, np.uint8)), dev.put(np.zeros_like(seen["q"]))
        ctx.paged_attention(out, heads * 64, dev.put(seen["q"]), heads * 64, kind, c, b, spec, work, n)
        assert np.count_nonzero(dev.get(work, (n // 4,), np.uint32) != 0xFFFFFFFF) >= 2 * 2 * len(long) * kv_heads      # maxima and sums of two parts of each at least
    check_attention(dev, rng, cache, kind, heads, kv_heads, 64, 16, lens.tolist(), new.tolist(), pad=2, sinks=True, edit=edit)


@pytest.mark.parametrize("cache", [F16, BF16, Q8, Q4], **KINDS)
def test_attention_of_large_scores(dev, cache):
    """one key takes nearly all weight: 2^-100 and less for the others"""
    check_attention(dev, np.random.default_rng(38), cache, F32, 2, 1, 128, 16, [200, 77], [3, 77], spread=60)


@pytest.mark.parametrize("kind", [F32, BF16], **KINDS)
@pytest.mark.parametrize("cache", [Q8, Q4], **KINDS)
def test_attention_of_large_and_small_scales(dev, kind, cache):
    """blocks next to the largest number that they can hold beside such of 10^-6"""
    def edit(pool, step):
        rng = np.random.default_rng(1)
        for p in range(90):
            page, at = step.place(pool, 0, p)
            pool.put(page, 0, 1, at, rng.standard_normal(64) * np.repeat([20000, 1e-6], 32)[::1 if p % 3 else -1])
            pool.put(page, 0, 0, at, rng.standard_normal(64) * np.repeat([1e-4, 0.1], 32))
    check_attention(dev, np.random.default_rng(44), cache, kind, 2, 1, 64, 16, [90], [20], edit=edit)


@pytest.mark.parametrize("kind", [F32, F16, BF16], **KINDS)
@pytest.mark.parametrize("cache", [F16, BF16], **KINDS)
def test_attention_of_numbers_that_are_not_finite(dev, kind, cache):
    """they show in rows that see them and in no others: in keys and values behind a row's position, and in what earlier users left in a page"""
    def edit(pool, step):
        for b, p, which, at, x in [(0, 30, 1, 3, np.inf), (0, 33, 1, 3, np.nan), (0, 35, 1, 40, -np.inf), (0, 36, 0, 0, np.nan), (1, 69, 1, 7, np.inf), (1, 5, 1, 8, -np.inf)]:
            page, i = step.place(pool, b, p)
            codes, _ = pool.row(page, 0, which, i)
            codes.view(np.uint16)[at] = ref.encode(np.float32([x]), pool.kind).view(np.uint16)[0]
    got, want = check_attention(dev, np.random.default_rng(39), cache, kind, 2, 1, 64, 16, [40, 70], [40, 2], edit=edit)
    assert np.isfinite(want[:30]).all() and np.isinf(want[30]).any() and np.isnan(want[36:40]).any()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("cache,kind", [(F16, F16), (F16, BF16), (BF16, BF16)], ids=lambda k: ref.NAMES[k])
def test_attention_of_numbers_that_are_not_finite_in_chunks(dev, cache, kind, dim):
    def edit(pool, step):
        for b, p, which, at, x in [(0, 30, 1, 3, np.inf), (0, 70, 1, 3, np.nan), (0, 71, 1, 40, -np.inf), (0, 75, 0, 0, np.nan), (1, 209, 1, 7, np.inf), (1, 5, 1, 8, -np.inf),
                                   (1, 190, 1, 63, np.nan)]:
            page, i = step.place(pool, b, p)
            codes, _ = pool.row(page, 0, which, i)
            codes.view(np.uint16)[at] = ref.encode(np.float32([x]), pool.kind).view(np.uint16)[0]
    got, want = check_attention(dev, np.random.default_rng(45), cache, kind, 2, 1, dim, 16, [80, 210], [80, 45], edit=edit)
    assert np.isfinite(want[:30]).all() and np.isinf(want[30]).any() and np.isnan(want[75:80]).any()


@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("cache,kind", [(F16, F16), (F16, BF16), (BF16, BF16), (F16, F32), (BF16, F32)], ids=lambda k: ref.NAMES[k])
@pytest.mark.parametrize("dim,new", [(64, 90), (128, 90), (64, 2), (128, 2), (32, 90)])
@pytest.mark.parametrize("keys", [330, 1100])      # one launch; cut into parts that a second one puts together
def test_attention_of_values_that_are_not_finite_and_weigh_next_to_nothing(dev, cache, kind, dim, new, keys, sinks):
    """An infinity times a weight is infinite, however small the weight is: it shows as itself in every row that sees it.  The first keys' scores are 200 below the others' (weights of
    e^-200, which 64 bits hold and 32 do not), some of the later ones' 25 (2^-36: 0 as fp16); with a learned logit 300 above all of them every weight is e^-300 or less."""
    rng = np.random.default_rng(63)
    pool = ref.Pool(cache, 1, dim, 16, keys // 16 + 3, rng)
    step = ref.Step(pool, [keys], [new], rng)
    unit = 8.0 / dim                      # of a key: a score of 1 with queries of 1 and a scale of 0.125
    far, some = 140, (150, 177, 200, 233)
    for p in range(keys):
        at = step.place(pool, 0, p)
        pool.put(at[0], 0, 0, at[1], np.full(dim, unit * (-200 if p < far else -25 if p in some else 0)) + rng.standard_normal(dim) * 0.01)
        v = rng.standard_normal(dim)
        for d, x in {7: {0: np.inf}, 100: {0: np.inf, 1: -np.inf, 2: np.inf}, 139: {3: -np.inf, 4: np.nan}, 150: {5: np.inf, 6: -np.inf}, 200: {6: np.inf}, 233: {2: -np.inf, 7: np.nan}}.get(p, {}).items():
            v[d] = x
        pool.put(at[0], 0, 1, at[1], v)
    s = np.array([300, 0], dtype=np.float32) if sinks else None
    got, held = run_attention(dev, pool, step, np.ones((new, 2, dim)), kind, 2, 0.125, 0, 0, s)
    want, size, reach, seen, mass = ref.attention(pool, step, held, 2, 0.125, 0, 0, s)
    assert np.isposinf(want[..., [0, 5]]).all() and np.isneginf(want[..., [1, 3]]).all() and np.isnan(want[..., [2, 4, 6, 7]]).all() and np.isfinite(want[..., 8:]).all()
    assert np.array_equal(got[..., :8], want[..., :8], equal_nan=True)
    bound = ref.attention_bound(want[..., 8:], size[..., 8:], reach, seen, mass[..., 8:], dim, kind, cache)
    assert np.all(np.abs(got[..., 8:] - want[..., 8:]) <= bound)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("cache,kind,window", [(F16, F16, 0), (BF16, BF16, 0), (F16, BF16, 700), (Q8, F16, 0)], ids=str)
def test_attention_of_a_chunk_behind_a_long_context(dev, cache, kind, window, dim):
    """few tiles of many keys: cut into parts"""
    check_attention(dev, np.random.default_rng(46), cache, kind, 4, 1, dim, 128, [1900, 333], [41, 10], window=window, sinks=True, pad=2)


def test_attention_of_chunks_without_pages(dev):
    def edit(pool, step):
        step.table[0, 2] = pool.pages
        step.table[0, 5] = NO_PAGE
        step.table[1, :] = 0xFFFFFF00
        step.lens[2] = 30                   # fewer than the new ones
    for sinks in (False, True):
        got, want = check_attention(dev, np.random.default_rng(47), F16, F16, 2, 2, 64, 16, [130, 50, 70], [90, 40, 70], sinks=sinks, edit=edit)
        assert not got[90:130].any() and not got[130:170].any() and got[170:].any() and got[:90].any()


@pytest.mark.parametrize("cache", [F16, BF16], **KINDS)
def test_attention_of_chunks_of_large_scores(dev, cache):
    """the reference of a row's weights is moved often, and by a lot"""
    check_attention(dev, np.random.default_rng(48), cache, BF16 if cache == BF16 else F16, 2, 1, 128, 16, [300, 177], [200, 177], spread=40)


@pytest.mark.parametrize("scale", [-0.2, 0.0])
@pytest.mark.parametrize("new", [1, 60])
def test_attention_scales(dev, scale, new):
    rng = np.random.default_rng(49)
    pool = ref.Pool(F16, 1, 64, 16, 12, rng)
    step = ref.Step(pool, [150], [new], rng)
    for p in range(150):
        at = step.place(pool, 0, p)
        for which in (0, 1):
            pool.put(at[0], 0, which, at[1], rng.standard_normal(64))
    got, held = run_attention(dev, pool, step, rng.standard_normal((new, 2, 64)), F16, 2, scale)
    want, size, reach, seen, mass = ref.attention(pool, step, held, 2, float(np.float32(scale)))
    assert np.all(np.abs(got - want) <= ref.attention_bound(want, size, reach, seen, mass, 64, F16, F16))


@pytest.mark.parametrize("cache,kind,new", [(BF16, F32, 1), (BF16, F32, 40), (BF16, BF16, 1), (BF16, BF16, 60)], ids=str)
@pytest.mark.parametrize("keys", [100, 600])
def test_attention_of_scores_far_below_zero(dev, cache, kind, new, keys):
    """Scores of -10^33 and less: the largest key's has all the weight, 10^27 above the next, so a row is its values, rounded at most twice (pieces, and the quotient)"""
    rng = np.random.default_rng(53)
    pool = ref.Pool(cache, 1, 64, 16, 40, rng)
    step = ref.Step(pool, [keys], [new], rng)
    v = ref.decode(ref.encode(rng.standard_normal((keys, 64)), BF16), BF16)
    best = rng.integers(0, keys - new)
    for p in range(keys):
        at = step.place(pool, 0, p)
        pool.put(at[0], 0, 0, at[1], np.full(64, 1e15 if p == best else 1.5e15 + 1e13 * (p % 90)))
        pool.put(at[0], 0, 1, at[1], v[p])
    got, held = run_attention(dev, pool, step, np.full((new, 2, 64), -1e17), kind, 2, 0.125)
    assert np.all(np.abs(got - v[best]) <= 2.0 ** -20 * np.abs(v[best]) if kind == F32 else got == v[best])


@pytest.mark.parametrize("cache", [F16, Q4], **KINDS)
@pytest.mark.parametrize("new", [2, 50])
def test_attention_of_sequences_that_share_pages(dev, cache, new):
    """a common beginning is stored once: the same pages in several rows of the table, and one sequence twice"""
    def edit(pool, step):
        step.table[1, :25] = step.table[0, :25]
        step.table[2] = step.table[0]
        step.lens[2] = step.lens[0]
    check_attention(dev, np.random.default_rng(54), cache, F16, 4, 2, 64, 16, [500, 470, 500], [new, new, new], edit=edit)


@pytest.mark.parametrize("cache,kind", [(F16, F16), (Q8, BF16), (BF16, F32)], ids=str)
@pytest.mark.parametrize("window,chunk,sinks", [(5, 0, True), (300, 0, False), (0, 50, False), (0, 400, True), (333, 256, True)], ids=str)
def test_attention_masks_of_calls_that_are_cut(dev, cache, kind, window, chunk, sinks):
    check_attention(dev, np.random.default_rng(55), cache, kind, 4, 2, 64, 16, [700, 450, 33], [2, 1, 3], window=window, chunk=chunk, sinks=sinks)
    check_attention(dev, np.random.default_rng(56), cache, kind, 4, 2, 64, 32, [700, 450], [40, 70], window=window, chunk=chunk, sinks=sinks)


@pytest.mark.parametrize("cache,kind", [(F16, F16), (Q4, BF16), (F16, F32)], ids=str)
@pytest.mark.parametrize("new", [1, 3])
def test_attention_of_many_heads_over_one(dev, cache, kind, new):
    """a token's heads fill more than a tile: tiles begin in the middle of a token"""
    check_attention(dev, np.random.default_rng(57), cache, kind, 150, 1, 64, 16, [500, 20, 3], [new, 2, 0], sinks=True, pad=1)


def test_a_table_without_columns(dev):
    """no position has a page: nothing is written or read back, and every row is 0"""
    lva, ctx = dev.lva, dev.ctx
    rng = np.random.default_rng(58)
    pool = ref.Pool(F16, 1, 64, 16, 4, rng)
    dpool, c = dev.cache(pool)
    b = lva.PagedBatch(1, 5, dev.put(np.array([0, 5], np.uint32)).value, dev.put(np.array([5], np.uint32)).value, None, 0)
    x = dev.put(rng.standard_normal((5, 64)).astype(np.float16))
    y = np.full((5, 64), 7.5, np.float16)
    out, dk = dev.put(y), dev.put(y)
    ctx.paged_write(c, b, x, 64, x, 64, F16)
    ctx.paged_read(c, b, dk, 64, dk, 64, F16)
    ctx.paged_attention(out, 64, x, 64, F16, c, b, lva.PagedAttnSpec(1, 0.1, 0, 0, None))
    assert np.array_equal(dev.get(dpool, pool.bytes.shape, np.uint8), pool.bytes) and np.array_equal(dev.get(dk, y.shape, np.float16), y)
    assert not dev.get(out, y.shape, np.float16).any()


def test_attention_of_more_workgroups_than_a_launch_has(dev):
    """refused before anything is looked at"""
    lva, ctx = dev.lva, dev.ctx
    p = dev.put(np.zeros(64, np.uint32))
    c = lva.PagedCache(p.value, F16, 64, 32, 16, 1)
    b, spec = lva.PagedBatch(1, (1 << 24) - 1, p.value, p.value, p.value, 1), lva.PagedAttnSpec(64, 1.0, 0, 0, None)
    with pytest.raises(lva.LvError, match="tokens"):
        ctx.paged_attention(p, 2048, p, 2048, F16, c, b, spec, p, 1 << 40)


@pytest.mark.parametrize("cache", [F16, Q8], **KINDS)
def test_attention_without_pages(dev, cache):
    """keys whose page is not in the pool are hidden; a row that sees nothing is 0, also beside a sink"""
    def edit(pool, step):
        step.table[0, 1] = pool.pages
        step.table[0, 3] = NO_PAGE
        step.table[1, :] = 0xFFFFFF00
        step.lens[2] = 2                    # fewer tokens than new ones: the first three are at positions before 0
    for sinks in (False, True):
        got, want = check_attention(dev, np.random.default_rng(40), cache, F16, 2, 2, 64, 16, [70, 20, 5], [30, 4, 5], sinks=sinks, edit=edit)
        assert not got[30:34].any() and not got[34:37].any() and got[37:].any()


def test_attention_beyond_the_table(dev):
    """a length that the table does not cover: what has no page is hidden"""
    def edit(pool, step):
        step.lens[0] = 4000
    check_attention(dev, np.random.default_rng(41), F16, F16, 2, 1, 64, 16, [64, 10], [6, 1], edit=edit, window=3980)


def test_attention_of_a_pool_beyond_32_bits(dev):
    """pages on either side of 4 GiB from the pool's start"""
    lva, ctx = dev.lva, dev.ctx
    rng = np.random.default_rng(42)
    small = ref.Pool(F16, 2, 128, 16, 8, rng)
    small.bytes[:] = ref.encode(rng.standard_normal(small.bytes.nbytes // 2), F16).view(np.uint8).reshape(small.bytes.shape)
    pages = (5 << 30) // (2 * small.block)
    big = ctx.alloc(pages * 2 * small.block)
    dev.held.append(big)
    step = ref.Step(small, [100], [3], rng)
    where = {p: at for p, at in zip(range(8), (0, 1, pages // 2, pages - 1, (1 << 32) // (2 * small.block) - 1, (1 << 32) // (2 * small.block), pages - 2, 7))}
    for p, at in where.items():
        lva.check(ctx.lib.lv_dev_upload(ctx.h, big.value + at * 2 * small.block, small.bytes[p].ctypes.data_as(C.c_void_p), 2 * small.block))
    q = ref.encode(rng.standard_normal((3, 4, 128)), F16)
    want, size, reach, seen, mass = ref.attention(small, step, ref.decode(q, F16), 4, 0.1)
    step.table = np.where(step.table < 8, np.vectorize(lambda p: where.get(int(p), 0))(step.table), step.table).astype(np.uint32)
    c = lva.PagedCache(big.value, F16, 2, 128, 16, pages)
    b = dev.batch(step)
    spec = lva.PagedAttnSpec(4, 0.1, 0, 0, None)
    n = ctx.paged_attention_workspace(F16, c, b, spec)
    out = dev.put(np.zeros((3, 512), np.float16))
    ctx.paged_attention(out, 512, dev.put(q), 512, F16, c, b, spec, dev.put(np.zeros(n + 16, np.uint8)), n)
    got = dev.get(out, (3, 4, 128), np.float16).astype(np.float64)
    assert np.all(np.abs(got - want) <= ref.attention_bound(want, size, reach, seen, mass, 128, F16, F16))
    k = dev.put(np.zeros((3, 256), np.float32))
    ctx.paged_read(c, b, k, 256, dev.put(np.zeros((3, 256), np.float32)), 256, F32)
    back = dev.get(k, (3, 2, 128), np.float32)
    for row, _, pos in step.rows():
        page = [p for p, at in where.items() if at == step.table[0, pos // 16]][0]
        for h in range(2):
            assert np.array_equal(back[row, h], small.get(page, h, 0, pos % 16))


def test_attention_workspace_refusals(dev):
    lva, ctx = dev.lva, dev.ctx
    rng = np.random.default_rng(43)
    pool = ref.Pool(F16, 1, 64, 16, 40, rng)
    step = ref.Step(pool, [100], [1], rng)
    _, c = dev.cache(pool)
    b, spec = dev.batch(step), lva.PagedAttnSpec(2, 0.1, 0, 0, None)
    assert ctx.paged_attention_workspace(F16, c, b, spec) == 0      # a table of so few positions is not cut
    b = dev.batch(ref.Step(pool, [500], [1], rng))
    n = ctx.paged_attention_workspace(F16, c, b, spec)
    assert n > 0
    p = dev.put(np.zeros((2, 128), np.float16))
    work = dev.put(np.zeros(n + 16, np.uint8))
    for w, size in ((None, n), (work, n - 1), (work.value + 8, n)):
        with pytest.raises(lva.LvError, match="workspace"):
            ctx.paged_attention(p, 128, p, 128, F16, c, b, spec, w, size)
    # nothing to do
    step = ref.Step(pool, [5], [0], rng)
    b = dev.batch(step)
    assert ctx.paged_attention_workspace(F16, c, b, spec) == 0
    ctx.paged_attention(None, 0, None, 0, F16, c, b, spec)
    ctx.paged_write(c, b, None, 0, None, 0, F16)
    ctx.paged_read(c, b, None, 0, None, 0, F16)


# ---- verification ------------------------------------------------------------------------------------------------------------------
def probabilities(rng, shape, spread=3.0):
    x = rng.standard_normal(shape) * spread
    p = np.exp(x - x.max(-1, keepdims=True))
    return (p / p.sum(-1, keepdims=True)).astype(np.float32)


def run_verify(dev, target, draft, tokens, counts, uniforms, pad=3):
    lva, ctx = dev.lva, dev.ctx
    seqs, drafts = tokens.shape
    vocab = target.shape[2]

    def wide(a):
        out = np.full((*a.shape[:-1], vocab + pad), 1e9, dtype=np.float32)      # what lies behind a row has no part in it
        out[..., :vocab] = a
        return dev.put(out).value
    b = lva.DraftBatch(seqs, drafts, vocab, wide(target), vocab + pad, wide(draft) if draft is not None else None, vocab + pad, dev.put(tokens.astype(np.uint32)).value,
                       dev.put(counts.astype(np.uint32)).value if counts is not None else None, dev.put(uniforms.astype(np.float32)).value)
    n = ctx.verify_drafts_workspace(b)
    work = dev.put(np.full(n + 64, 0xFF, np.uint8))
    t, a = dev.put(np.full((seqs + 1, drafts + 1), 77, np.uint32)), dev.put(np.full(seqs + 1, 77, np.uint32))
    ctx.verify_drafts(t, a, b, work, n)
    t, a = dev.get(t, (seqs + 1, drafts + 1), np.uint32), dev.get(a, (seqs + 1,), np.uint32)
    assert np.all(t[seqs] == 77) and a[seqs] == 77 and np.all(dev.get(work, (n + 64,), np.uint8)[n:] == 0xFF)
    return t[:seqs], a[:seqs]


@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("seqs,drafts,vocab", [(1, 1, 1), (3, 2, 2), (1, 4, 32000), (40, 7, 513), (9, 64, 100), (2, 3, 128256), (5, 5, 2049), (70, 1, 256), (300, 2, 513), (16, 1, 32768),
                                               (17, 1, 16385), (1, 2, 33001)])
def test_verify(dev, seqs, drafts, vocab, sampled):
    rng = np.random.default_rng(51)
    target = probabilities(rng, (seqs, drafts + 1, vocab))
    draft = probabilities(rng, (seqs, drafts, vocab)) * 0.3 + target[:, :drafts] * np.float32(0.7)
    tokens = np.array([[rng.choice(vocab, p=r.astype(np.float64) / r.astype(np.float64).sum()) for r in s] for s in draft])
    uniforms = rng.random((seqs, drafts + 1)).astype(np.float32)
    uniforms[uniforms >= 1] = 0
    for counts in (None, rng.integers(0, drafts + 2, seqs)):
        got = run_verify(dev, target, draft if sampled else None, tokens, counts, uniforms)
        want = ref.verify(target, draft if sampled else None, tokens, counts if counts is not None else np.full(seqs, drafts), uniforms)
        assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])


@pytest.mark.parametrize("vocab", [500, 40000])      # one launch, two
@pytest.mark.parametrize("drafts", [63, 64])
def test_verify_drafts_that_all_stand(dev, drafts, vocab):
    """as many drafts as a wave has lanes, none of them refused: the next token is from the row behind them"""
    rng = np.random.default_rng(65)
    target = probabilities(rng, (2, drafts + 1, vocab))
    draft = target[:, :drafts].copy()
    tokens = np.array([[rng.choice(vocab, p=r.astype(np.float64) / r.astype(np.float64).sum()) for r in s] for s in draft])
    uniforms = np.minimum(rng.random((2, drafts + 1)).astype(np.float32), np.float32(0.99999))
    draft[1, drafts - 1] = 0              # the second sequence's last one is one that the draft never gives: it stands too
    got = run_verify(dev, target, draft, tokens, None, uniforms)
    want = ref.verify(target, draft, tokens, np.full(2, drafts), uniforms)
    assert np.all(want[1] == drafts) and np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])
    target[0, drafts - 1, int(tokens[0, drafts - 1])] = 0      # the very last one refused
    got = run_verify(dev, target, draft, tokens, None, uniforms)
    want = ref.verify(target, draft, tokens, np.full(2, drafts), uniforms)
    assert want[1].tolist() == [drafts - 1, drafts] and np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])


def test_verify_borders(dev):
    """random numbers at their ends, weights of 0 at a row's ends and in its middle, rows without weight, drafts outside the vocabulary, NaN"""
    rng = np.random.default_rng(52)
    V, top = 5000, np.nextafter(np.float32(1), np.float32(0))
    target, draft = np.zeros((12, 3, V), np.float32), np.zeros((12, 2, V), np.float32)
    tokens, uniforms = np.zeros((12, 2), np.int64), np.full((12, 3), 0.5, np.float32)
    target[:, :, 100:4900] = probabilities(rng, (12, 3, 4800))
    draft[:, :, 200:300] = 0.01
    tokens[:] = 250
    uniforms[0] = 0                       # the first token with weight, no draft refused that the target can give
    uniforms[1] = (top, top, top)         # the last one with weight
    tokens[2, 1] = V                      # outside
    tokens[3, 0] = 0xFFFFFFFF
    draft[4] = target[4, :2]              # the same: stands whatever the number is
    uniforms[4, :2] = top
    target[5] = 0                         # no weight at all: refused, token 0
    target[6, 0] = 0
    target[6, 0, 4000] = 1
    draft[6, 0] = target[6, 0]
    tokens[6, 0] = 17                     # refused (0 < 0 is not), and nothing left: from the target
    target[7, 0, ::3] = np.nan
    draft[7, 0, 1::3] = np.nan
    tokens[7, 0] = 102                    # NaN
    target[8, 0] = -target[8, 0]
    draft[9, 0] = 1                       # more than the target everywhere
    tokens[9, 0] = 4000
    uniforms[9] = (0.9, 0.9, 0)
    target[10, 0, 4999] = 0.25            # the very last entry
    uniforms[10] = (top, 0.1, top)
    draft[10, 0, 250] = 1
    target[11, 0, 250] = np.inf
    got = run_verify(dev, target, draft, tokens, None, uniforms)
    want = ref.verify(target, draft, tokens, np.full(12, 2), uniforms)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])
    got = run_verify(dev, target, None, tokens, None, uniforms)
    want = ref.verify(target, None, tokens, np.full(12, 2), uniforms)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])


def test_verified_tokens_follow_the_target(dev):
    """what speculative sampling is for: whatever the drafts' distribution, a first token comes out as often as the target says.  20000 draws from 6 tokens:
    the largest deviation allowed is 5 standard deviations, 5 sqrt(p (1 - p) / 20000)"""
    rng = np.random.default_rng(53)
    n, target, draft = 20000, np.float32([0.05, 0.3, 0.0, 0.4, 0.15, 0.1]), np.float32([0.4, 0.1, 0.2, 0.1, 0.1, 0.1])
    tokens = rng.choice(6, (n, 1), p=draft.astype(np.float64) / draft.astype(np.float64).sum())
    uniforms = np.minimum(rng.random((n, 2)).astype(np.float32), np.nextafter(np.float32(1), np.float32(0)))
    got, _ = run_verify(dev, np.broadcast_to(target, (n, 2, 6)), np.broadcast_to(draft, (n, 1, 6)), tokens, None, uniforms, pad=0)
    p = target.astype(np.float64)
    assert np.all(np.abs(np.bincount(got[:, 0], minlength=6) / n - p) <= 5 * np.sqrt(p * (1 - p) / n))


def test_verify_workspace_refusals(dev):
    lva, ctx = dev.lva, dev.ctx
    p = dev.put(np.zeros(4096, np.float32))
    assert ctx.verify_drafts_workspace(lva.DraftBatch(1, 1, 1000, p.value, 1000, None, 0, p.value, None, p.value)) == 0      # one launch
    b = lva.DraftBatch(1, 1, 40000, p.value, 40000, None, 0, p.value, None, p.value)
    n = ctx.verify_drafts_workspace(b)
    for w, size in ((None, n), (p, n - 1), (p.value + 8, n)):
        with pytest.raises(lva.LvError, match="workspace"):
            ctx.verify_drafts(p, p, b, w, size)
    with pytest.raises(lva.LvError, match="null"):
        ctx.verify_drafts(None, p, b, p, n)
    none = lva.DraftBatch(0, 1, 1000, None, 1000, None, 0, None, None, None)
    assert ctx.verify_drafts_workspace(none) == 0
    ctx.verify_drafts(None, None, none, None, 0)


# ---- together ----------------------------------------------------------------------------------------------------------------------
class Graph:
    """a captured graph of what `calls` puts on the context's stream"""

    def __init__(self, ctx, calls):
        self.hip, self.ctx, self.stream = C.CDLL("libamdhip64.so"), ctx, C.c_void_p(ctx.stream())
        graph, self.exe = C.c_void_p(), C.c_void_p()
        assert self.hip.hipStreamBeginCapture(self.stream, 2) == 0      # relaxed: this thread only
        calls()
        assert self.hip.hipStreamEndCapture(self.stream, C.byref(graph)) == 0
        assert self.hip.hipGraphInstantiate(C.byref(self.exe), graph, None, None, C.c_size_t(0)) == 0
        assert self.hip.hipGraphDestroy(graph) == 0

    def launch(self):
        assert self.hip.hipGraphLaunch(self.exe, self.stream) == 0

    def close(self):
        assert self.hip.hipGraphExecDestroy(self.exe) == 0


@pytest.mark.parametrize("columns", [12, 30])      # one launch of attention and of verification; two of each
@pytest.mark.parametrize("cache,kind", [(F16, F32), (BF16, BF16), (Q8, F16), (Q4, BF16)], ids=lambda k: ref.NAMES[k])
def test_a_step_of_drafts_captured_and_replayed(dev, cache, kind, columns):
    """Queries and keys turned, rows written, attention over all of it, drafts verified: one graph, replayed for several steps whose lengths, pages, rows and random
    numbers change on the device.  Every step against the definitions, on the pool as the device has it."""
    lva, ctx = dev.lva, dev.ctx
    rng = np.random.default_rng(61)
    heads, kv_heads, dim, page, seqs, drafts, vocab = 8, 2, 64, 16, 3, 3, 700 if columns == 12 else 33000
    new = drafts + 1
    pool = ref.Pool(cache, kv_heads, dim, page, 40, rng)
    table = np.full((seqs, columns), NO_PAGE, dtype=np.uint32)
    table[:, :12] = rng.permutation(40)[:36].reshape(seqs, 12)
    lens = np.array([0, 20, 100])
    for s in range(seqs):                 # what the sequences hold already
        for p in range(lens[s]):
            for h in range(kv_heads):
                for which in (0, 1):
                    pool.put(table[s, p // page], h, which, p % page, rng.standard_normal(dim))
    rows, width = seqs * new, (heads + 2 * kv_heads) * dim
    dpool, c = dev.cache(pool)
    starts = (np.arange(seqs + 1) * new).astype(np.uint32)
    dlens, dpos, dqkv = dev.put(np.zeros(seqs, np.uint32)), dev.put(np.zeros(rows, np.uint32)), dev.put(ref.encode(np.zeros((rows, width)), kind))
    b = lva.PagedBatch(seqs, rows, dev.put(starts).value, dlens.value, dev.put(table).value, columns)
    spec, rot = lva.PagedAttnSpec(heads, 0.125, 0, 0, None), lva.RotateSpec(dim, 1e4, (0, 0, 0), lva.ROTATE_HALVES)
    n = ctx.paged_attention_workspace(kind, c, b, spec)
    assert (n > 0) == (columns > 24)
    work = dev.put(np.zeros(n + 16, np.uint8))
    out = dev.put(ref.encode(np.zeros((rows, heads * dim)), kind))
    size = ref.BYTES[kind]
    dt, dd, dx, du = (dev.put(np.zeros(s, t)) for s, t in (((seqs, new, vocab), np.float32), ((seqs, drafts, vocab), np.float32), ((seqs, drafts), np.uint32), ((seqs, new), np.float32)))
    db = lva.DraftBatch(seqs, drafts, vocab, dt.value, vocab, dd.value, vocab, dx.value, None, du.value)
    m = ctx.verify_drafts_workspace(db)
    vwork, dtok, dacc = dev.put(np.zeros(m + 16, np.uint8)), dev.put(np.zeros((seqs, new), np.uint32)), dev.put(np.zeros(seqs, np.uint32))

    def calls():
        ctx.rotate(dqkv, width, dqkv, width, kind, dpos, rows, heads + kv_heads, dim, rot)
        ctx.paged_write(c, b, dqkv.value + heads * dim * size, width, dqkv.value + (heads + kv_heads) * dim * size, width, kind)
        ctx.paged_attention(out, heads * dim, dqkv, width, kind, c, b, spec, work, n)
        ctx.verify_drafts(dtok, dacc, db, vwork, m)

    graph = Graph(ctx, calls)
    other = dev.put(np.zeros(1 << 20, np.uint8))
    for turn in range(5):
        lens = lens + new
        qkv = ref.encode(rng.standard_normal((rows, width)) * 1.5, kind)
        pos = np.concatenate([np.arange(x - new, x) for x in lens]).astype(np.uint32)
        target = probabilities(rng, (seqs, new, vocab))
        draft = (probabilities(rng, (seqs, drafts, vocab)) + target[:, :drafts]) / 2
        tokens = np.array([[rng.choice(vocab, p=r.astype(np.float64) / r.astype(np.float64).sum()) for r in s] for s in draft]).astype(np.uint32)
        uniforms = np.minimum(rng.random((seqs, new)).astype(np.float32), np.float32(0.99999))
        for p, a in ((dlens, lens.astype(np.uint32)), (dpos, pos), (dqkv, qkv), (dt, target), (dd, draft), (dx, tokens), (du, uniforms)):
            a = np.ascontiguousarray(a)
            lva.check(ctx.lib.lv_dev_upload(ctx.h, p, a.ctypes.data_as(C.c_void_p), a.nbytes))
        if turn == 0:
            calls()                       # the eager step first, on the same inputs as the first replay
            eager = [dev.get(p, (rows, heads * dim), ref.DTYPE[kind]) for p in (out,)][0], dev.get(dtok, (seqs, new), np.uint32)
            lva.check(ctx.lib.lv_dev_upload(ctx.h, dqkv, qkv.ctypes.data_as(C.c_void_p), qkv.nbytes))
        graph.launch()
        got, turned = dev.get(out, (rows, heads * dim), ref.DTYPE[kind]), dev.get(dqkv, (rows, width), ref.DTYPE[kind])
        tok, acc = dev.get(dtok, (seqs, new), np.uint32), dev.get(dacc, (seqs,), np.uint32)
        if turn == 0:
            assert np.array_equal(got, eager[0]) and np.array_equal(tok, eager[1])
        # rotation
        x = ref.decode(qkv, kind).reshape(rows, -1, dim)
        want, reach = ref.rotate(x[:, :heads + kv_heads], pos[None], dim, 1e4, halves=True)
        y = ref.decode(turned, kind).reshape(rows, -1, dim)
        assert np.all(np.abs(y[:, :heads + kv_heads] - want) <= 2e-6 * reach + HALF_STEP[kind] * np.abs(want) + (2.0 ** -24 if kind == F16 else 0))
        assert np.array_equal(y[:, heads + kv_heads:], x[:, heads + kv_heads:])
        # rows, from what was turned
        step = ref.Step.__new__(ref.Step)
        step.lens, step.new, step.pad, step.table, step.starts, step.tokens = lens, np.full(seqs, new), 0, table, starts, rows
        for row, s, p in step.rows():
            at = step.place(pool, s, p)
            for h in range(kv_heads):
                pool.put(at[0], h, 0, at[1], y[row, heads + h])
                pool.put(at[0], h, 1, at[1], y[row, heads + kv_heads + h])
        assert np.array_equal(dev.get(dpool, pool.bytes.shape, np.uint8), pool.bytes)
        # attention
        want, size_, reach, seen, mass = ref.attention(pool, step, y[:, :heads], heads, 0.125)
        assert np.all(np.abs(ref.decode(got, kind).reshape(want.shape) - want) <= ref.attention_bound(want, size_, reach, seen, mass, dim, kind, cache))
        # drafts
        w = ref.verify(target, draft, tokens, np.full(seqs, drafts), uniforms)
        assert np.array_equal(tok, w[0]) and np.array_equal(acc, w[1])
        lva.check(ctx.lib.lv_dev_zero(ctx.h, other, 1 << 20))      # other work between the replays
        lens = lens - (drafts - acc.astype(np.int64))              # refused drafts' rows are written over by the next step
    graph.close()


@pytest.mark.parametrize("cache,kind", [(F16, F32), (BF16, BF16), (Q8, BF16), (Q4, F16)], ids=lambda k: ref.NAMES[k])
@pytest.mark.parametrize("lens,new", [([1500, 400, 90], [1, 3, 1]), ([1500, 400], [200, 70]), ([300], [300])], ids=str)
def test_calls_repeat_themselves(dev, cache, kind, lens, new):
    """the same call ten times, other work between: the same bits"""
    lva, ctx = dev.lva, dev.ctx
    rng = np.random.default_rng(66)
    pool = ref.Pool(cache, 2, 128, 16, 140, rng)
    pool.bytes[:] = rng.integers(0, 48, pool.bytes.shape, dtype=np.uint8)      # small finite numbers and scales
    step = ref.Step(pool, lens, new, rng)
    _, c = dev.cache(pool)
    b, spec = dev.batch(step), lva.PagedAttnSpec(8, 0.01, 0, 0, None)
    q = dev.put(ref.encode(rng.standard_normal((step.tokens, 1024)), kind))
    n = ctx.paged_attention_workspace(kind, c, b, spec)
    work, out = dev.put(np.full(n + 16, 0xFF, np.uint8)), dev.put(np.zeros((step.tokens, 1024), ref.DTYPE[kind]))
    first = None
    for turn in range(10):
        lva.check(ctx.lib.lv_dev_zero(ctx.h, out, step.tokens * 1024 * ref.BYTES[kind]))
        ctx.paged_attention(out, 1024, q, 1024, kind, c, b, spec, work, n)
        got = dev.get(out, (step.tokens, 1024 * ref.BYTES[kind]), np.uint8)
        first = got if first is None else first
        assert first.any() and np.array_equal(got, first), turn


def test_two_contexts_at_once(lva, ctx, dev):
    """calls of two contexts overlap, each with a workspace of its own; results are those of a call alone, bit for bit"""
    rng = np.random.default_rng(62)
    pool = ref.Pool(Q8, 2, 128, 16, 130, rng)
    step = ref.Step(pool, [1500, 400], [1, 1], rng)
    pool.bytes[:] = rng.integers(0, 48, pool.bytes.shape, dtype=np.uint8)      # scales up to 0.11
    _, c = dev.cache(pool)
    b, spec = dev.batch(step), lva.PagedAttnSpec(8, 0.01, 0, 0, None)
    q = dev.put(ref.encode(rng.standard_normal((2, 1024)), F16))
    n = ctx.paged_attention_workspace(F16, c, b, spec)
    second = lva.Context(0)
    outs = [dev.put(np.zeros((2, 1024), np.float16)) for _ in range(3)]
    works = [dev.put(np.zeros(n + 16, np.uint8)) for _ in range(3)]
    ctx.paged_attention(outs[2], 1024, q, 1024, F16, c, b, spec, works[2], n)
    ctx.sync()
    for _ in range(20):
        for i, x in enumerate((ctx, second)):
            x.paged_attention(outs[i], 1024, q, 1024, F16, c, b, spec, works[i], n)
    second.sync()
    first, other, alone = (dev.get(p, (2, 1024), np.uint16) for p in outs)
    assert np.array_equal(first, alone) and np.array_equal(other, alone) and alone.any()
    second.close()
