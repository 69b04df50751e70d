"""Attention over the key/value cache (KVCache.attend) where values are infinite, scores are large, or a token's neighbours in the
call change: the kernels of few and of many rows against plain implementations in 64 bits (kv_reference.py)."""
import math

import pytest
import torch

from kv_reference import attend as ref_attend, held
from qwen3_tts_rs_amd import KVCache
from test_gpu_kv_cache import bounds, rand, table_of, workspace

pytestmark = pytest.mark.gpu


def cache_with(k, v, fmt="bf16", page=64):
    """One sequence of the given keys and values on shuffled pages: the cache and a function (new, ctx) -> batch."""
    n, kv, d = k.shape
    table, pages = table_of([n], page)
    cache = KVCache(pages=pages, kv_heads=kv, head_dim=d, format=fmt, page_tokens=page)
    cache.write(0, cache.batch([n], [n], table), k, v)
    return cache, lambda new, ctx: cache.batch([new], [ctx], table)


# --------------------------------------------------------------------------------------------------------------- infinities
def check_infinite(out, q, k, v, scale, window=0):
    """Rows that see an infinity: the formula's infinities and NaN (of both signs: NaN); every other element within its bound."""
    e = ref_attend(q, k.double(), v.double(), scale, window)
    got = out.double().cpu()
    assert torch.equal(got.isnan(), e.isnan())
    assert torch.equal(got.isinf(), e.isinf()) and torch.equal(got[e.isinf()], e[e.isinf()])
    # the bound of the finite elements: without the infinities, none of which a row with a finite element of that column sees
    clean = v.double().cpu().nan_to_num(0, 0, 0)
    tol = bounds(q, k.double(), clean, scale, window, e.nan_to_num(0, 0, 0))
    assert ((got - e).abs() <= tol)[e.isfinite()].all()


@pytest.mark.parametrize("window", [0, 20])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,new", [(1, 9), (3, 9), (2, 70), (2, 200), (5, 300)])
def test_infinite_values_from_the_first_key_on(heads, new, dim, window):
    """A prompt from nothing: infinities among the first keys a tile sees, where no maximum is known yet, and in every block after."""
    k, v, q = rand((new, 1, dim), 1), rand((new, 1, dim), 2), rand((new, heads, dim), 3)
    for i, at in enumerate(range(0, new, 13)):
        v[at, 0, (3 * i) % dim] = math.inf if i % 3 else -math.inf
    v[3, 0, 5], v[5, 0, 5] = math.inf, -math.inf  # both signs: NaN for the rows that see both
    cache, batch = cache_with(k, v)
    check_infinite(cache.attend(0, batch(new, new), q, window=window), q, k, v, dim ** -0.5, window)


@pytest.mark.parametrize("new", [128, 127, 30, 15])
@pytest.mark.parametrize("ctx", [700, 1040, 1100, 1290, 1601, 2070])
def test_infinite_values_where_a_part_begins(ctx, new):
    """Parts of the key range that begin among the chunk's own keys, which some of its rows see and others do not."""
    d, heads = 128, 1
    k, v, q = rand((ctx, 1, d), 1), rand((ctx, 1, d), 2), rand((new, heads, d), 3)
    for i, back in enumerate((1, 20, 41, 62, 83, 104, 125)):
        v[ctx - back, 0, 7 * i] = math.inf
    v[10, 0, 100] = -math.inf  # seen by all
    cache, batch = cache_with(k, v)
    b = batch(new, ctx)
    check_infinite(cache.attend(0, b, q), q, k, v, d ** -0.5)


@pytest.mark.parametrize("heads,new", [(1, 16), (1, 30), (1, 130), (4, 130)])
def test_infinite_values_beside_a_maximum_that_jumps(heads, new):
    """The first 64 keys score about 320 below the others (2^-460 of their weights): the infinity stands beside the higher ones."""
    d, ctx = 64, 130
    k, v, q = rand((ctx, 1, d), 1), rand((ctx, 1, d), 2), rand((new, heads, d), 3)
    q[:, :, 0] = 16
    k[:, :, 0] = 0
    k[:64, :, 0] = -160
    v[100, 0, 9], v[117, 0, 30] = math.inf, -math.inf
    cache, batch = cache_with(k, v)
    check_infinite(cache.attend(0, batch(new, ctx), q), q, k, v, d ** -0.5)
# ------------------------------------------------------------------------------------------------------------- large scores
@pytest.mark.parametrize("top", [1e7, 1e9, 1e10, 1e12, 1e20, 1e30, 1e37])
@pytest.mark.parametrize("heads,new,ctx", [(1, 1, 150), (1, 5, 150), (8, 4, 150), (40, 5, 150), (2, 150, 150), (3, 60, 900), (1, 1, 3000), (5, 5, 3000), (1, 40, 3000)])
def test_large_finite_scores(heads, new, ctx, top):
    """Scores of up to `top`: one product of two bf16 numbers each, exact in f32.  Two of them that differ do so by 2^-8 of the
    larger, 2^15 and more, so that every weight but the largest is zero (or the same, where scores are the same) and the f32
    rounding of a score does not count: what is left of the bound is the rounding of weights and output and the sums.  Every third
    token's scores are ordinary ones, below 8."""
    d = 64
    k, v = torch.zeros(ctx, 1, d), rand((ctx, 1, d), 2)
    k[:, 0, 0] = torch.randint(-255, 256, (ctx,), generator=torch.Generator().manual_seed(5)).float() / 256
    k = k.to(torch.bfloat16).cuda()
    q = rand((new, heads, d), 3)
    small = torch.arange(new) % 3 == 2
    # scale 2^40 at the top end: raw scores stay below the largest f32
    scale = 2.0 ** -3 if top < 1e20 else 2.0 ** 40
    q[:, :, 0] = 2.0 ** math.floor(math.log2(top / scale))
    q[small, :, 0] = 8.0 / scale
    cache, batch = cache_with(k, v)
    out = cache.attend(0, batch(new, ctx), q, scale=scale).double().cpu()
    e = ref_attend(q, k.double(), v.double(), scale)
    a = ref_attend(q, k.double(), v.double().abs(), scale)
    assert e.isfinite().all()
    # z = 8 in the bound of the ordinary tokens (bounds() in test_gpu_kv_cache.py)
    tol = 1.01 * (2.0 ** -8 * e.abs() + (2.0 ** -8 + 2 * (d + 4) * 2.0 ** -24 * 8 + (ctx + 100) * 2.0 ** -23) * a)
    assert ((out - e).abs() <= tol).all(), float(((out - e).abs() / tol).nan_to_num(1e9).max())


@pytest.mark.parametrize("heads", [1, 40])
def test_scores_that_overflow_as_products_with_the_scale(heads):
    """Finite q k whose product with the scale is not: +infinity, so the row is NaN as with an infinite q k, whatever the kernel."""
    d, ctx = 64, 70
    k, v, q = torch.zeros(ctx, 1, d, dtype=torch.bfloat16, device="cuda"), rand((ctx, 1, d), 2), rand((2, heads, d), 3)
    q[:, :, 0] = 2.0 ** 60
    k[5, 0, 0] = 2.0 ** 20
    cache, batch = cache_with(k, v)
    b = batch(2, ctx)
    assert cache.attend(0, b, q, scale=2.0 ** 50).isnan().all()
    out = cache.attend(0, b, q, scale=2.0 ** 40)  # 2^120: the one key
    assert torch.equal(out, v[5].expand(2, heads, d))


# ------------------------------------------------------------------------------------------------------ neighbours in a call
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_prompt_in_two_parts_gives_the_same(dim, fmt, window):
    """The last tokens of a prompt get bit for bit what they get when the first ones come in a call before: a row's result depends on
    its own scores alone, not on which rows share its tile (one part of the keys in all calls)."""
    n, heads = 300, 4
    k, v, q = rand((n, 2, dim), 1), rand((n, 2, dim), 2), rand((n, heads, dim), 3, scale=4.0)
    cache, batch = cache_with(k, v, fmt)
    assert workspace(cache, batch(n, n), heads, window) == 0
    whole = cache.attend(0, batch(n, n), q, window=window)
    for cut in (1, 7, 64, 100, 203, 259):
        assert torch.equal(cache.attend(0, batch(n - cut, n), q[cut:], window=window), whole[cut:]), cut
        assert torch.equal(cache.attend(0, batch(cut, cut), q[:cut], window=window), whole[:cut]) or 2 * cut <= 32, cut
