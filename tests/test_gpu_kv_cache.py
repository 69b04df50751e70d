"""Key/value cache and attention over it (KVCache) on the GPU against plain implementations in 64 bits (kv_reference.py).

What the cache holds is compared exactly.  Attention in bf16 is off by at most
    2^-8 |o|                    its own rounding,
    2^-8 A                      the rounding of the probabilities, A = sum_j p_j |v_j|,
    (2 (d + 4) 2^-24 Z + (c + 100) 2^-23) A
                                f32 scores with Z = max_j scale sum |q k_j| (an error x of a score moves its probability by x, and the
                                sum that divides it as much), exponentials and sums over c keys,
with the products of these terms below a hundredth of them: bounds() adds them up per element.
"""
import ctypes as C
import math

import pytest
import torch

from kv_reference import attend as ref_attend, held
from qwen3_tts_rs_amd import KVBatch, KVCache, QttsError, _lib

pytestmark = pytest.mark.gpu
FMTS = ["bf16", "e4m3", "int8"]


def same(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def table_of(ctx, page, spare=3, seed=0):
    """Shuffled pages for sequences of the given lengths, -1 behind them: (n_seq, max_pages), pages in all."""
    need = [-(-c // page) for c in ctx]
    perm = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    t = torch.full((len(ctx), max(need + [1])), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for i in range(n):
            t[b, i] = perm.pop()
    return t.cuda(), sum(need) + spare


def rand(shape, seed, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def split(x, lens):
    return list(torch.split(x.cpu(), lens))


def bounds(q, k, v, scale, window, exact, holes=None):
    """See the module's docstring; q (n, heads, d), k, v (ctx, kv, d) held values."""
    n, heads, d = q.shape
    a = ref_attend(q, k, v.abs(), scale, window, holes)
    z = scale * float((q.double().abs().cpu().amax((0, 1)) @ k.double().abs().cpu().nan_to_num(0, 0, 0).amax((0, 1))))
    return 1.01 * (2.0 ** -8 * exact.abs() + (2.0 ** -8 + 2 * (d + 4) * 2.0 ** -24 * z + (k.shape[0] + 100) * 2.0 ** -23) * a)


def check_attend(out, q, keys, values, new, ctx, fmt, scale, window=0, holes=None):
    outs, qs, ks, vs = split(out, new), split(q, new), split(keys, ctx), split(values, ctx)
    for b in range(len(new)):
        if new[b] == 0:
            continue
        k, v = held(ks[b], fmt), held(vs[b], fmt)
        hb = holes[b] if holes else None
        e = ref_attend(qs[b], k, v, scale, window, hb)
        tol = bounds(qs[b], k, v, scale, window, e, hb)
        got = outs[b].double()
        bad = ~((got - e).abs() <= tol) & ~((got == e) | (got.isnan() & e.isnan()))
        assert not bad.any(), (b, new[b], ctx[b], float(((got - e).abs() / tol).nan_to_num(1e9).max()), bad.nonzero()[:3].tolist())


# ---------------------------------------------------------------------------------------------------- writing and reading
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt", FMTS)
def test_write_and_read_back(fmt, dtype, dim):
    for kv, page, new, ctx in ((1, 16, [1], [1]), (3, 16, [5, 0, 1, 33], [5, 7, 40, 33]), (8, 64, [70, 2], [200, 130]), (2, 1024, [1, 17], [9, 17])):
        table, pages = table_of(ctx, page)
        cache = KVCache(pages=pages, kv_heads=kv, head_dim=dim, format=fmt, layers=2, page_tokens=page)
        old = [c - n for c, n in zip(ctx, new)]
        k, v = rand((sum(ctx), kv, dim), 1, dtype, 3.0), rand((sum(ctx), kv, dim), 2, dtype)
        ks, vs = split(k, ctx), split(v, ctx)
        part = lambda xs, lo: torch.cat([x[:o] if lo else x[o:] for x, o in zip(xs, old)]).cuda()  # noqa: E731
        cache.write(1, cache.batch(old, old, table), part(ks, True), part(vs, True))
        cache.write(1, cache.batch(new, ctx, table), part(ks, False), part(vs, False))
        got = cache.read(1, cache.batch(ctx, ctx, table), dtype=torch.float32)
        assert same(got[0], held(k.cpu(), fmt)) and same(got[1], held(v.cpu(), fmt))
        got = cache.read(1, cache.batch(new, ctx, table))  # bf16 holds what 8 bits stand for exactly
        assert same(got[0], held(part(ks, False).cpu(), fmt)) and same(got[1], held(part(vs, False).cpu(), fmt))
        other = cache.read(0, cache.batch(ctx, ctx, table), dtype=torch.float32)
        assert not other[0].any() and not other[1].any()  # the other layer still holds zeros
        assert cache.bytes() >= 2 * 2 * pages * page * kv * dim


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_blocks_that_are_hard_to_hold(fmt):
    x = rand((40, 2, 64), 3, torch.float32)
    x[0] = 0
    x[1, :, :32] = 448.0
    x[2, :, :32] = 127.0 * 2.0 ** 9
    x[3, :, 5] = math.inf
    x[4, :, 40] = -math.inf
    x[5, :, 63] = math.nan
    x[6] *= 1e-38   # among them values below the smallest normal f32
    x[7] *= 2.0 ** -112
    x[8] *= 1e37
    x[9, :, ::2] *= 1e-9
    x[10, :, :32] = torch.arange(32).float().cuda() * 2.0 ** -10 + 448.0 - 31 * 2.0 ** -10
    x[11, :, 0], x[11, :, 1:] = 127.0, torch.arange(63).float().cuda() + 0.5  # halves: to even
    x[12, :, 0], x[12, :, 1:] = 448.0, 2.0 ** -10 * (torch.arange(63).float().cuda() + 0.5)
    x[13, :, 0] = torch.finfo(torch.float32).max
    table, pages = table_of([40], 16)
    cache = KVCache(pages=pages, kv_heads=2, head_dim=64, format=fmt, page_tokens=16)
    b = cache.batch([40], [40], table)
    cache.write(0, b, x, -x)
    k, v = cache.read(0, b, dtype=torch.float32)
    for t in range(40):
        assert same(k[t], held(x[t].cpu(), fmt)) and same(v[t], held(-x[t].cpu(), fmt)), t


@pytest.mark.parametrize("fmt", FMTS)
def test_layouts_of_the_tensors(fmt):
    """Heads first, slices of a wider projection, a broadcast token: any strides whose rows start at multiples of 16 bytes."""
    kv, d, n = 2, 64, 37
    table, pages = table_of([n], 16)
    cache = KVCache(pages=pages, kv_heads=kv, head_dim=d, format=fmt, page_tokens=16)
    b = cache.batch([n], [n], table)
    heads_first = rand((kv, n, d), 4).transpose(0, 1)
    wide = rand((n, 3 * kv * d + 8), 5)[:, 8:].unflatten(1, (3 * kv, d))[:, kv:2 * kv]
    cache.write(0, b, heads_first, wide)
    out_k, out_v = torch.zeros(kv, n, d, device="cuda"), torch.full((n, 2 * kv, d), 7.0, device="cuda")
    cache.read(0, b, out=(out_k.transpose(0, 1), out_v[:, kv:]))
    assert same(out_k.transpose(0, 1), held(heads_first.cpu(), fmt)) and same(out_v[:, kv:], held(wide.cpu(), fmt)) and (out_v[:, :kv] == 7).all()
    one = rand((1, 1, d), 6).expand(n, kv, d)
    cache.write(0, b, one, one)
    q = rand((kv * 2, n, d), 7).transpose(0, 1)
    out = torch.zeros(n, kv * 4, d, dtype=torch.bfloat16, device="cuda")[:, ::2]
    got = cache.attend(0, b, q, out=out)
    assert got is out
    check_attend(out, q, one, one, [n], [n], fmt, d ** -0.5)


def test_holes_are_neither_written_nor_read():
    page, d = 16, 64
    ctx = [50, 33]
    table, pages = table_of(ctx, page, spare=0)
    cache = KVCache(pages=pages, kv_heads=1, head_dim=d, format="e4m3", page_tokens=page)
    whole = cache.batch(ctx, ctx, table)
    k, v = rand((83, 1, d), 1), rand((83, 1, d), 2)
    cache.write(0, whole, k, v)
    holed = table.clone()
    holed[0, 1], holed[1, 0] = -7, pages  # below and just above the range
    hb = cache.batch(ctx, ctx, holed)
    gk, gv = cache.read(0, hb)
    ek, ev = held(k.cpu(), "e4m3"), held(v.cpu(), "e4m3")
    for e in (ek, ev):
        e[16:32], e[50:66] = 0, 0
    assert same(gk, ek) and same(gv, ev)
    cache.write(0, hb, k * 2, v * 2)
    gk, _ = cache.read(0, whole)
    ek = held(k.cpu() * 2, "e4m3")
    ek[16:32], ek[50:66] = held(k.cpu(), "e4m3")[16:32], held(k.cpu(), "e4m3")[50:66]
    assert same(gk, ek)


# ----------------------------------------------------------------------------------------------------------- attention
SHAPES = [  # heads, kv heads, head_dim, page, new, ctx
    (1, 1, 64, 16, [1], [1]),
    (2, 1, 64, 64, [1, 1, 1], [1, 16, 17]),
    (16, 8, 128, 64, [1, 1], [113, 300]),
    (5, 1, 128, 16, [1, 3, 0, 2], [64, 65, 9, 2]),
    (16, 1, 64, 32, [1], [129]),
    (40, 2, 64, 16, [1, 2], [31, 200]),
    (3, 3, 64, 64, [16, 15], [16, 400]),
    (4, 2, 128, 64, [33, 8], [33, 200]),
    (2, 2, 128, 16, [63, 64, 65, 129], [63, 64, 65, 129]),
    (6, 2, 64, 16, [100, 1, 43], [257, 64, 44]),
    (8, 1, 128, 128, [50], [191]),
]


@pytest.mark.parametrize("window", [0, 1, 20, 64])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("fmt", FMTS)
def test_attend(fmt, shape, window):
    heads, kv, d, page, new, ctx = SHAPES[shape]
    table, pages = table_of(ctx, page, seed=shape)
    cache = KVCache(pages=pages, kv_heads=kv, head_dim=d, format=fmt, page_tokens=page)
    k, v, q = rand((sum(ctx), kv, d), 1), rand((sum(ctx), kv, d), 2), rand((sum(new), heads, d), 3)
    cache.write(0, cache.batch(ctx, ctx, table), k, v)
    b = cache.batch(new, ctx, table)
    scale = None if shape % 2 else 0.3
    out = cache.attend(0, b, q, scale=scale, window=window)
    check_attend(out, q, k, v, new, ctx, fmt, scale or d ** -0.5, window)
    assert torch.equal(out, cache.attend(0, b, q, scale=scale, window=window))


@pytest.mark.parametrize("heads,new", [(1, 1), (4, 9), (2, 80)])
@pytest.mark.parametrize("fmt", FMTS)
def test_long_contexts_are_cut_into_parts(fmt, heads, new):
    """One sequence and kv head: the keys are walked in parts that a second launch joins; a ragged companion has one part."""
    d, page, ctx = 128, 64, [5003, 100]
    table, pages = table_of(ctx, page)
    cache = KVCache(pages=pages, kv_heads=1, head_dim=d, format=fmt, page_tokens=page)
    k, v, q = rand((sum(ctx), 1, d), 1), rand((sum(ctx), 1, d), 2), rand((2 * new, heads, d), 3, scale=2.0)
    cache.write(0, cache.batch(ctx, ctx, table), k, v)
    for window in (0, 2500):
        b = cache.batch([new, new], ctx, table)
        assert workspace(cache, b, heads, window) > 0
        check_attend(cache.attend(0, b, q, window=window), q, k, v, [new, new], ctx, fmt, d ** -0.5, window)


def workspace(cache, b, heads, window=0):
    n = C.c_int64(-1)
    _lib.check(cache.lib.qtts_kv_attend_workspace(cache._kv, b._ptr, heads, window, C.byref(n)))
    return n.value


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("new", [1, 6, 70])
def test_what_is_masked_may_hold_anything(fmt, new):
    """NaN and infinities behind the sequence, before the window, in holes and in later tokens of the chunk reach no row that does not
    see them; rows that see them get what the formula gives."""
    d, page, ctx, window = 64, 16, 150, 40
    table, pages = table_of([ctx + 20], page)
    cache = KVCache(pages=pages, kv_heads=2, head_dim=d, format=fmt, page_tokens=page)
    k, v, q = rand((ctx + 20, 2, d), 1), rand((ctx + 20, 2, d), 2), rand((new, 4, d), 3)
    k[ctx:], v[ctx:] = math.nan, math.inf                 # behind the sequence
    k[:20], v[:20] = math.nan, -math.inf                  # before every window
    hole = range(112, 128)
    k[112:128], v[112:128] = math.inf, math.nan           # a hole
    if new > 1:
        k[ctx - 1, 0], v[ctx - 2, 1, 5] = math.nan, math.inf  # the chunk's last tokens
        v[ctx - 3, 0, 7] = -math.inf
    cache.write(0, cache.batch([ctx + 20], [ctx + 20], table), k, v)
    table[0, 7] = -1
    out = cache.attend(0, cache.batch([new], [ctx], table), q, window=window)
    e = ref_attend(q, held(k[:ctx].cpu(), fmt), held(v[:ctx].cpu(), fmt), d ** -0.5, window, set(hole))
    if new > 6:
        assert e[:new - 3].isfinite().all()  # only the last rows see what is not finite
    got = out.double().cpu()
    assert torch.equal(got.isnan(), e.isnan()) and torch.equal(got.isinf(), e.isinf())
    check_attend(out, q, k[:ctx], v[:ctx], [new], [ctx], fmt, d ** -0.5, window, holes=[set(hole)])


def test_rows_that_see_nothing_are_zero():
    d, page = 64, 16
    table = torch.tensor([[-1, 0], [1, -1]], dtype=torch.int32, device="cuda")
    cache = KVCache(pages=2, kv_heads=1, head_dim=d, format="bf16", page_tokens=page)
    k = rand((40, 1, d), 1)
    cache.write(0, cache.batch([20, 20], [20, 20], table), k, k)
    for heads, new in ((2, 20), (10, 20)):  # both kernels
        q = rand((2 * new, heads, d), 2)
        out = cache.attend(0, cache.batch([new, new], [20, 20], table), q, window=4)
        check_attend(out, q, k, k, [new, new], [20, 20], "bf16", d ** -0.5, 4, holes=[set(range(16)), set(range(16, 20))])
        assert not out[:16].any() and out[16:20].any()


def test_arrays_that_break_their_bounds_stay_inside():
    """Lengths beyond the host bounds are cut and pages outside the cache are holes; rows no sequence owns stay as they are."""
    d, page = 64, 16
    cache = KVCache(pages=4, kv_heads=1, head_dim=d, format="int8", page_tokens=page)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    k = rand((6, 1, d), 1)
    big = 2 ** 31 - 1
    for start, ctx, table in ((i32(0, 3, 6), i32(big, -big), i32(0, 1, 2, 3)), (i32(-big, big, big), i32(32, 32), i32(big, -big, 4, -1)),
                              (i32(5, 2, -1), i32(3, 4), i32(0, 1, 2, 3)), (i32(0, 1, 2), i32(0, 0), i32(0, 1, 2, 3))):
        b = KVBatch(start, ctx, table.view(2, 2), 6, 3, 32)
        out = torch.full((6, 20, d), 7.0, dtype=torch.bfloat16, device="cuda")
        cache.write(0, b, k, k)
        gk, _ = cache.read(0, b, out=(torch.full_like(k, 7.0), torch.full_like(k, 7.0)))
        for heads in (1, 20):
            cache.attend(0, b, rand((6, heads, d), 2), out=out[:, :heads])
            assert not out.isnan().any()
    torch.cuda.synchronize()
    b = KVBatch(i32(0, 2, 3), i32(2, 1), i32(0, 1, 2, 3).view(2, 2), 6, 2, 32)
    cache.write(0, b, k, k)
    out = torch.full((6, 2, d), 7.0, dtype=torch.bfloat16, device="cuda")
    rk, rv = torch.full_like(k, 7.0), torch.full_like(k, 7.0)
    cache.attend(0, b, rand((6, 2, d), 2), out=out)
    cache.read(0, b, out=(rk, rv))
    assert (out[3:] == 7).all() and (rk[3:] == 7).all() and (rv[3:] == 7).all() and (out[:3] != 7).any()


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_offsets_beyond_32_bits(fmt):
    """Pages whose elements lie more than 2^32 elements (and bytes) into the cache."""
    d, kv, page = 128, 8, 64
    pages = 33000  # x 2 x 8 x 64 x 128 = 4.3e9 elements
    cache = KVCache(pages=pages, kv_heads=kv, head_dim=d, format=fmt, page_tokens=page)
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    k, v, q = rand((150, kv, d), 1), rand((150, kv, d), 2), rand((150, kv, d), 3)
    b = cache.batch([150], [150], table)
    cache.write(0, b, k, v)
    gk, gv = cache.read(0, b)
    assert same(gk, held(k.cpu(), fmt)) and same(gv, held(v.cpu(), fmt))
    check_attend(cache.attend(0, b, q), q, k, v, [150], [150], fmt, d ** -0.5)
    one = cache.batch([1], [150], table)
    check_attend(cache.attend(0, one, q[:1]), q[:1], k, v, [1], [150], fmt, d ** -0.5)


# ------------------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("fmt", FMTS)
def test_a_serving_loop(fmt):
    """Two layers: prompts in parts of odd lengths, single tokens, drafted tokens of which some are dropped, a sequence that goes and
    one that takes its pages."""
    heads, kv, d, page, layers = 4, 2, 128, 16, 2
    cache = KVCache(pages=40, kv_heads=kv, head_dim=d, format=fmt, layers=layers, page_tokens=page)
    free = list(range(40))
    seqs = {}  # name: dict(pages, k, v per layer)

    def step(parts, drop=None, seed=0):
        names = list(parts)
        for s in names:
            q = seqs.setdefault(s, dict(pages=[], k=[torch.zeros(0, kv, d)] * layers, v=[torch.zeros(0, kv, d)] * layers))
            while len(q["pages"]) * page < len(q["k"][0]) + parts[s]:
                q["pages"].append(free.pop(0))
        width = max(len(seqs[s]["pages"]) for s in names)
        table = [seqs[s]["pages"] + [-1] * (width - len(seqs[s]["pages"])) for s in names]
        new = [parts[s] for s in names]
        ctx = [len(seqs[s]["k"][0]) + parts[s] for s in names]
        b = cache.batch(new, ctx, table)
        for layer in range(layers):
            k, v, q = (rand((sum(new), h, d), seed * 31 + layer * 7 + i) for i, h in enumerate((kv, kv, heads)))
            cache.write(layer, b, k, v)
            out = cache.attend(layer, b, q)
            for s, x, y in zip(names, split(k, new), split(v, new)):
                seqs[s]["k"][layer], seqs[s]["v"][layer] = torch.cat([seqs[s]["k"][layer], x]), torch.cat([seqs[s]["v"][layer], y])
            check_attend(out, q, torch.cat([seqs[s]["k"][layer] for s in names]), torch.cat([seqs[s]["v"][layer] for s in names]), new, ctx, fmt, d ** -0.5)
        for s, n in (drop or {}).items():
            for x in ("k", "v"):
                seqs[s][x] = [t[:len(t) - n] for t in seqs[s][x]]

    step({"a": 37, "b": 5}, seed=1)
    step({"a": 80, "b": 1, "c": 21}, seed=2)
    for i in range(3):
        step({"a": 1, "b": 1, "c": 1}, seed=3 + i)
    step({"a": 5, "c": 5}, drop={"a": 3, "c": 5}, seed=7)
    step({"a": 1, "b": 1, "c": 5}, drop={"c": 2}, seed=8)
    free[:0] = seqs.pop("a")["pages"]  # reused first, with what they hold
    step({"d": 50, "b": 1, "c": 1}, seed=9)


def test_shared_pages():
    """Sequences that share a prompt's pages and go on on pages of their own."""
    heads, kv, d, page = 2, 1, 64, 16
    cache = KVCache(pages=8, kv_heads=kv, head_dim=d, format="int8", page_tokens=page)
    k, v = rand((32, kv, d), 1), rand((32, kv, d), 2)
    cache.write(0, cache.batch([32], [32], [[3, 5]]), k, v)
    table = [[3, 5, 0], [3, 5, 1], [3, 5, 2]]
    new, ctx = [3, 1, 9], [35, 33, 41]
    b = cache.batch(new, ctx, table)
    nk, nv, q = rand((13, kv, d), 3), rand((13, kv, d), 4), rand((13, heads, d), 5)
    cache.write(0, b, nk, nv)
    join = lambda x, y: torch.cat([torch.cat([x.cpu(), p]) for p in split(y, new)])  # noqa: E731
    check_attend(cache.attend(0, b, q), q, join(k, nk), join(v, nv), new, ctx, "int8", d ** -0.5)


# ------------------------------------------------------------------------------------------------- streams and graphs
def test_another_stream_and_the_current_device():
    d, ctx = 128, 2000
    table, pages = table_of([ctx], 64)
    cache = KVCache(pages=pages, kv_heads=1, head_dim=d, format="e4m3")
    k, v, q = rand((ctx, 1, d), 1), rand((ctx, 1, d), 2), rand((1, 2, d), 3)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        cache.write(0, cache.batch([ctx], [ctx], table), k, v)
        out = cache.attend(0, cache.batch([1], [ctx], table), q)
    s.synchronize()
    assert torch.cuda.current_device() == 0
    check_attend(out, q, k, v, [1], [ctx], "e4m3", d ** -0.5)


def test_captured_steps():
    """A decode step (write and attend) captured twice over two caches; lengths move on in place between replays; both graphs run
    side by side with eager work between them."""
    heads, kv, d, page, n = 4, 2, 64, 16, 3
    most = 1200
    loops = []
    for g, fmt in enumerate(("int8", "bf16")):
        ctx = [700 + 10 * g, 5, 300]
        table, pages = table_of([most] * n, page, seed=g)
        cache = KVCache(pages=pages, kv_heads=kv, head_dim=d, format=fmt, page_tokens=page)
        k, v = rand((sum(ctx), kv, d), 10 + g), rand((sum(ctx), kv, d), 20 + g)
        cache.write(0, cache.batch(ctx, ctx, table), k, v)
        lens = torch.tensor(ctx, dtype=torch.int32, device="cuda")
        b = KVBatch(torch.arange(n + 1, dtype=torch.int32, device="cuda"), lens, table, n, 1, most)
        assert workspace(cache, b, heads) > 0
        bufs = [torch.zeros(n, h, d, dtype=torch.bfloat16, device="cuda") for h in (kv, kv, heads)]
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            lens += 1
            cache.write(0, b, bufs[0], bufs[1])
            out = cache.attend(0, b, bufs[2])
        loops.append(dict(cache=cache, b=b, fmt=fmt, bufs=bufs, graph=graph, out=out, ctx=ctx, ks=split(k, ctx), vs=split(v, ctx), lens=lens))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(4):
        for g, w in enumerate(loops):
            for j, buf in enumerate(w["bufs"]):
                buf.copy_(rand(buf.shape, 100 + 10 * i + 3 * g + j))
        torch.cuda.synchronize()
        for w, s in zip(loops, streams):
            with torch.cuda.stream(s):
                w["graph"].replay()
        torch.cuda.synchronize()
        for w in loops:
            w["ctx"] = [c + 1 for c in w["ctx"]]
            assert w["lens"].tolist() == w["ctx"]
            w["ks"] = [torch.cat([x, y]) for x, y in zip(w["ks"], split(w["bufs"][0], [1] * n))]
            w["vs"] = [torch.cat([x, y]) for x, y in zip(w["vs"], split(w["bufs"][1], [1] * n))]
            check_attend(w["out"], w["bufs"][2], torch.cat(w["ks"]), torch.cat(w["vs"]), [1] * n, w["ctx"], w["fmt"], d ** -0.5)
            assert torch.equal(w["out"], w["cache"].attend(0, w["b"], w["bufs"][2]))  # eager, between the replays


def test_two_threads():
    """Two host threads, each with a stream and batches of its own, on one cache."""
    import threading
    d, page = 64, 16
    cache = KVCache(pages=64, kv_heads=2, head_dim=d, format="e4m3", page_tokens=page)
    ctx = [300, 45]
    table = torch.arange(38, dtype=torch.int32, device="cuda").view(2, 19)
    data = [[rand((sum(ctx), 2, d), 10 * i + j) for j in range(2)] + [rand((2, 6, d), 10 * i + 5)] for i in range(2)]
    tables = [table, torch.stack([torch.arange(38, 57), torch.cat([torch.arange(57, 60), torch.full((16,), -1)])]).to(torch.int32).cuda()]
    outs, errors = [None, None], []
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    cache.write(0, cache.batch(ctx, ctx, tables[i]), data[i][0], data[i][1])
                    outs[i] = cache.attend(0, cache.batch([1, 1], ctx, tables[i]), data[i][2])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 - reported by the test
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for i in range(2):
        check_attend(outs[i], data[i][2], data[i][0], data[i][1], [1, 1], ctx, "e4m3", d ** -0.5)


@pytest.mark.parametrize("new", [1, 40])
def test_many_sequences_and_output_over_the_queries(new):
    """1500 sequences of a few tokens; the output takes the queries' place."""
    d, page, n = 64, 16, 1500
    ctx = [new + b % 7 for b in range(n)]
    table, pages = table_of(ctx, page)
    cache = KVCache(pages=pages, kv_heads=1, head_dim=d, format="int8", page_tokens=page)
    k, v, q = rand((sum(ctx), 1, d), 1), rand((sum(ctx), 1, d), 2), rand((n * new, 2, d), 3)
    cache.write(0, cache.batch(ctx, ctx, table), k, v)
    b = cache.batch([new] * n, ctx, table)
    out = cache.attend(0, b, q)
    place = q.clone()
    cache.attend(0, b, place, out=place)
    assert torch.equal(out, place)
    some = list(range(0, n, 97))
    pick = lambda x, lens: torch.cat([split(x, lens)[i] for i in some])  # noqa: E731
    check_attend(pick(out, [new] * n), pick(q, [new] * n), pick(k, ctx), pick(v, ctx), [new] * len(some), [ctx[i] for i in some], "int8", d ** -0.5)


def test_single_token_and_single_head_ignore_their_stride():
    """The stride of a dimension of one element is not used, whatever torch says it is."""
    d, page, ctx = 64, 16, 37
    table, pages = table_of([ctx], page)
    cache = KVCache(pages=pages, kv_heads=1, head_dim=d, page_tokens=page)
    k, v, q = rand((ctx, 1, d), 1), rand((ctx, 1, d), 2), rand((1, 1, d), 3)
    odd = lambda x: torch.as_strided(x, x.shape, (x.stride(0) if x.shape[0] > 1 else 3, 5, 1))  # noqa: E731
    cache.write(0, cache.batch([ctx], [ctx], table), odd(k), odd(v))
    b = cache.batch([1], [ctx], table)
    out = torch.empty_like(q)
    cache.attend(0, b, odd(q), out=odd(out))
    check_attend(out, q, k, v, [1], [ctx], "bf16", d ** -0.5)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("group,new", [(1, 17), (17, 1), (3, 7), (5, 5), (8, 4), (32, 1), (4, 8), (11, 3)])
def test_17_to_33_rows(group, new, fmt, dim):
    """Rows a kv head from just over 16 to just over 32: alone and with the keys in parts, with holes, with a window, an infinity in V that
    some rows see."""
    page, kv = 32, 2
    ctx, news = [1100, new, 333], [new, new, max(1, new - 1)]
    table, pages = table_of(ctx, page)
    cache = KVCache(pages=pages, kv_heads=kv, head_dim=dim, format=fmt, page_tokens=page)
    k, v, q = rand((sum(ctx), kv, dim), 1), rand((sum(ctx), kv, dim), 2), rand((sum(news), group * kv, dim), 3)
    cache.write(0, cache.batch(ctx, ctx, table), k, v)
    b = cache.batch(news, ctx, table)
    assert workspace(cache, b, group * kv) > 0
    check_attend(cache.attend(0, b, q), q, k, v, news, ctx, fmt, dim ** -0.5)
    check_attend(cache.attend(0, b, q, window=40), q, k, v, news, ctx, fmt, dim ** -0.5, 40)
    short = cache.batch([new], [new], table[1:2].contiguous())  # one part
    assert workspace(cache, short, group * kv) == 0
    sl = slice(ctx[0], ctx[0] + new)
    q1 = q[news[0]:news[0] + new].contiguous()
    check_attend(cache.attend(0, short, q1), q1, k[sl], v[sl], [new], [new], fmt, dim ** -0.5)
    if new > 2:  # the last token's value: only its own rows see it
        v[ctx[0] + new - 1, 0, 5] = float("inf")
        cache.write(0, cache.batch([1], [new], table[1:2].contiguous()), k[sl][-1:], v[sl][-1:])
        out = cache.attend(0, short, q1)
        assert out[:-1].isfinite().all() and not out[-1, :group].isfinite().all() and out[-1, group:].isfinite().all()
    table[0, 3], table[0, 30], table[2, 0] = -1, pages, -7
    holes = [set(range(96, 128)) | set(range(960, 992)), set(), set(range(32))]
    if new <= 2:
        check_attend(cache.attend(0, cache.batch(news, ctx, table), q), q, k, v, news, ctx, fmt, dim ** -0.5, 0, holes)


@pytest.mark.parametrize("heads", [1, 40])
def test_scores_that_are_not_finite(heads):
    """Overflowing scores: +infinity makes the row NaN, -infinity leaves the key without weight."""
    d, page, ctx = 64, 16, 70
    table, pages = table_of([ctx], page)
    cache = KVCache(pages=pages, kv_heads=1, head_dim=d, page_tokens=page)
    k, v, q = rand((ctx, 1, d), 1), rand((ctx, 1, d), 2), rand((2, heads, d), 3)
    q[:, :, 0] = 1e38
    k[:, :, 0] = 0
    k[3, 0, 0] = -1e38                     # -infinity for both rows
    cache.write(0, cache.batch([ctx], [ctx], table), k, v)
    b = cache.batch([2], [ctx], table)
    check_attend(cache.attend(0, b, q), q, k, v, [2], [ctx], "bf16", d ** -0.5)
    k[:, 0, 0] = -1e38                     # every score -infinity: no key has weight
    cache.write(0, cache.batch([ctx], [ctx], table), k, v)
    assert (cache.attend(0, b, q) == 0).all()
    k[:, 0, 0] = 0
    k[ctx - 1, 0, 0] = 1e38                # +infinity for the last row only
    cache.write(0, cache.batch([ctx], [ctx], table), k, v)
    out = cache.attend(0, b, q)
    assert out[1].isnan().all() and out[0].isfinite().all()


@pytest.mark.parametrize("fmt", FMTS)
def test_wide_tiles_in_parts_with_holes_and_a_window(fmt):
    """Row tiles whose keys are walked in parts (few kv heads, long contexts), ragged, with holes, with and without a window."""
    d, page, heads, kv = 128, 64, 6, 2
    ctx, new = [2600, 900, 70], [70, 45, 70]
    table, pages = table_of(ctx, page)
    cache = KVCache(pages=pages, kv_heads=kv, head_dim=d, format=fmt, page_tokens=page)
    k, v, q = rand((sum(ctx), kv, d), 1), rand((sum(ctx), kv, d), 2), rand((sum(new), heads, d), 3)
    cache.write(0, cache.batch(ctx, ctx, table), k, v)
    table[0, 3], table[0, 40], table[1, 0] = -1, pages, -5
    holes = [set(range(192, 256)) | set(range(2560, 2600)), set(range(64)), set()]
    b = cache.batch(new, ctx, table)
    assert workspace(cache, b, heads) > 0
    for window in (0, 1700):
        check_attend(cache.attend(0, b, q, window=window), q, k, v, new, ctx, fmt, d ** -0.5, window, holes)


# ------------------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    d = 64
    for bad in (dict(pages=0), dict(kv_heads=0), dict(head_dim=96), dict(layers=0), dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=2048)):
        with pytest.raises(QttsError):
            KVCache(**{**dict(pages=2, kv_heads=1, head_dim=d), **bad})
    with pytest.raises(QttsError):
        KVCache(pages=1 << 30, kv_heads=1024, head_dim=128, layers=1 << 20)
    cache = KVCache(pages=2, kv_heads=2, head_dim=d, format="int8", page_tokens=16)
    table = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    with pytest.raises(QttsError, match="new <= ctx"):
        cache.batch([3], [2], table)
    with pytest.raises(QttsError, match="longer than"):
        cache.batch([1], [33], table)
    b = cache.batch([2], [4], table)
    ok = rand((2, 2, d), 1)
    for k, v in ((ok[:1], ok), (ok, ok[:, :1]), (ok[..., :32], ok), (ok.half(), ok.half()), (ok, ok.float()), (ok.cpu(), ok),
                 (rand((2, 2, 2 * d), 1)[..., ::2], ok), (rand((2, 2 * d + 1), 1)[:, 1:].unflatten(1, (2, d)), ok)):
        with pytest.raises(QttsError):
            cache.write(0, b, k, v)
    with pytest.raises(QttsError, match="no such layer"):
        cache.write(1, b, ok, ok)
    with pytest.raises(QttsError, match="no such layer"):
        cache.read(1 << 32, b)
    with pytest.raises(QttsError, match="overlap"):
        cache.read(0, b, out=(torch.empty(1, 2, d, device="cuda").expand(2, 2, d), torch.empty(2, 2, d, device="cuda")))
    with pytest.raises(QttsError, match="overlap"):
        cache.attend(0, b, ok, out=torch.empty(2, 1, d, dtype=torch.bfloat16, device="cuda").expand(2, 2, d))
    for q, kw in ((rand((2, 3, d), 1), {}), (ok.float(), {}), (ok, dict(scale=0.0)), (ok, dict(scale=-1.0)), (ok, dict(scale=math.nan)),
                  (ok, dict(window=-1)), (ok.clone().requires_grad_(), {}), (ok, dict(out=ok[:1].clone()))):
        with pytest.raises(QttsError):
            cache.attend(0, b, q, **kw)
    far = KVBatch(b.q_start, b.ctx_len, table, 2, 2, 33)  # max_ctx beyond the table's columns
    with pytest.raises(QttsError, match="max_pages"):
        cache.attend(0, far, ok)
    with pytest.raises(QttsError, match="one tensor"):
        cache.read(0, b, out=(ok, ok))
    for kw in (dict(scale=1e31), dict(scale=math.inf), dict(window=-(1 << 40))):
        with pytest.raises(QttsError):
            cache.attend(0, b, ok, **kw)
    # a workspace that is too small
    long = KVCache(pages=64, kv_heads=1, head_dim=d, page_tokens=64)
    lb = long.batch([1], [4000], torch.arange(64, dtype=torch.int32, device="cuda").view(1, 64))
    need = workspace(long, lb, 1)
    assert need > 0
    q = rand((1, 1, d), 1)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    for ptr, n in ((ws.data_ptr(), need - 1), (None, need), (ws.data_ptr() + 8, need)):
        a = _lib.KvAttendArgs(q.data_ptr(), q.data_ptr(), d, d, d, d, 1, 1.0, 0, ptr, n)
        assert long.lib.qtts_kv_attend(long._kv, 0, lb._ptr, C.addressof(a), None) == -1
    cache.close()
    with pytest.raises(QttsError, match="closed"):
        cache.write(0, b, ok, ok)
    # nothing to do is no error
    empty = long.batch([], [], torch.empty(0, 4, dtype=torch.int32, device="cuda"))
    none = torch.empty(0, 1, d, dtype=torch.bfloat16, device="cuda")
    long.write(0, empty, none, none)
    assert long.attend(0, empty, none).shape == (0, 1, d) and long.read(0, empty)[0].shape == (0, 1, d)
    zero = long.batch([0], [5], torch.zeros(1, 1, dtype=torch.int32, device="cuda"))
    assert long.attend(0, zero, none).shape == (0, 1, d)
