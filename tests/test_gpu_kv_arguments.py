"""Arguments of the key/value cache's calls (KVCache) that are refused, and their neighbours that are not."""
import pytest
import torch

from kv_reference import held
from qwen3_tts_rs_amd import KVCache, QttsError
from test_gpu_kv_cache import check_attend, rand, same, table_of

pytestmark = pytest.mark.gpu


def _cache(n, kv, d, fmt="bf16"):
    table, pages = table_of([n], 16)
    cache = KVCache(pages=pages, kv_heads=kv, head_dim=d, format=fmt, page_tokens=16)
    k, v = rand((n, kv, d), 1), rand((n, kv, d), 2)
    b = cache.batch([n], [n], table)
    cache.write(0, b, k, v)
    return cache, b, k, v


def test_rows_read_into_one_buffer():
    n, kv, d = 20, 2, 64
    cache, b, k, v = _cache(n, kv, d, "int8")
    flat = torch.zeros(4 * n * kv * d, device="cuda")
    view = lambda at, ts=kv * d, hs=d: flat.as_strided((n, kv, d), (ts, hs, 1), at)  # noqa: E731
    for x, y in ((view(0), view(d)), (view(0), view(kv * d)), (view(0), view((n - 1) * kv * d)), (view(kv * d), view(0)), (view(0), view(4)),
                 (view(0, 2 * kv * d), view(0, 2 * kv * d, 2 * d)), (view(0, 2 * kv * d), view(kv * d // 2, 2 * kv * d))):
        with pytest.raises(QttsError, match="overlap|one tensor"):
            cache.read(0, b, out=(x, y))
    assert not flat.any()
    for x, y in ((view(0), view(n * kv * d)), (view(0, 2 * kv * d), view(kv * d, 2 * kv * d)), (view(0, 2 * kv * d, 2 * d), view(d, 2 * kv * d, 2 * d)),
                 (view(0, d, 2 * n * d), view(n * d, d, 2 * n * d))):
        flat.zero_()
        cache.read(0, b, out=(x, y))
        assert same(x, held(k.cpu(), "int8")) and same(y, held(v.cpu(), "int8"))


@pytest.mark.parametrize("heads", [2, 40])
def test_output_that_overlaps_the_queries(heads):
    n, d = 20, 64
    cache, b, k, v = _cache(n, 1, d)
    flat = rand((4 * n * heads * d,), 3)
    view = lambda at, ts=heads * d, hs=d: flat.as_strided((n, heads, d), (ts, hs, 1), at)  # noqa: E731
    for q, out in ((view(0), view(8)), (view(0), view(heads * d)), (view(heads * d), view(0)), (view(0), view(0, 2 * heads * d)),
                   (view(0), view(0, d, n * d)), (view(0, 2 * heads * d), view((heads - 1) * d, 2 * heads * d))):
        before = flat.clone()
        with pytest.raises(QttsError, match="overlaps q"):
            cache.attend(0, b, q, out=out)
        assert torch.equal(flat, before)
    with pytest.raises(QttsError, match="overlaps q"):  # one token for all, written over
        cache.attend(0, b, view(0, 0), out=view(0))
    for q, out in ((view(0), view(0)), (view(0), view(n * heads * d)), (view(0, 2 * heads * d), view(heads * d, 2 * heads * d)),
                   (view(0, d, 2 * n * d), view(n * d, d, 2 * n * d))):
        flat.copy_(rand(flat.shape, 4))
        keep = q.clone()
        cache.attend(0, b, q, out=out)
        check_attend(out, keep, k, v, [n], [n], "bf16", d ** -0.5)


def test_tensors_with_a_tangent():
    """Forward-mode differentiation: refused, as a tensor that requires a gradient is, instead of a result that has lost its tangent."""
    import torch.autograd.forward_ad as fwad
    n, d = 5, 64
    cache, b, k, v = _cache(n, 1, d)
    q = rand((n, 2, d), 3)
    with fwad.dual_level():
        for call in (lambda: cache.attend(0, b, fwad.make_dual(q, q)), lambda: cache.attend(0, b, q, out=fwad.make_dual(q.clone(), q)),
                     lambda: cache.write(0, b, fwad.make_dual(k, k), v), lambda: cache.write(0, b, k, fwad.make_dual(v, v)),
                     lambda: cache.read(0, b, out=(fwad.make_dual(k.clone(), k), v.clone()))):
            with pytest.raises(QttsError, match="tangent"):
                call()
        out = cache.attend(0, b, q)  # without one, inside the level
    check_attend(out, q, k, v, [n], [n], "bf16", d ** -0.5)


def test_a_step_of_no_sequences_from_host_numbers():
    """A serving loop whose sequences have all ended passes empty lists."""
    cache, _, k, _ = _cache(5, 1, 64)
    b = cache.batch([], [], [])
    none = k[:0]
    cache.write(0, b, none, none)
    assert cache.attend(0, b, none).shape == (0, 1, 64) and cache.read(0, b)[0].shape == (0, 1, 64)
    b = cache.batch([0, 0], [5, 0], [[0], [-1]])
    assert cache.attend(0, b, none).shape == (0, 1, 64)
