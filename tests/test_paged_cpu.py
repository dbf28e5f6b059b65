"""The paged KV cache without a GPU: shapes, argument checks and their status codes, and the
host side's pages (handed out, given back, refused)."""
import ctypes

import pytest

INVALID, MISALIGNED, UNSUPPORTED = -1, -2, -3


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.load_library()


def _cache(pkg, **kw):
    c = pkg.paged._PagedCacheC(num_pages=8, kv_heads=2, head_dim=128, page_size=16, max_seqs=2, max_pages=4, tier=0,
                               pages=256, scale=256, open=256, table=256)
    for k, v in kw.items():
        setattr(c, k, v)
    return ctypes.byref(c)


def _step(pkg, **kw):
    s = pkg.paged._PagedStepC(batch=1, rows=3, max_new=3, seq=256, start=256, length=256, cu=256)
    for k, v in kw.items():
        setattr(s, k, v)
    return ctypes.byref(s)


def test_cache_bytes(lib):
    # pages of codes, scales, two open blocks a sequence, the table; each rounded up to 256 bytes
    assert lib.ee_paged_cache_bytes(10, 8, 128, 16, 3, 5, 0) == 10 * 2 * 8 * 16 * 128 + 768 + 3 * 2 * 2 * 8 * 16 * 128 * 2 + 256
    assert lib.ee_paged_cache_bytes(10, 8, 128, 16, 3, 5, 2) == 2 * 10 * 2 * 8 * 16 * 128 + 256
    for bad in ((0, 8, 128, 16, 3, 5, 0), (10, 0, 128, 16, 3, 5, 0), (10, 8, 96, 16, 3, 5, 0), (10, 8, 128, 24, 3, 5, 0),
                (10, 8, 128, 256, 3, 5, 0), (10, 8, 128, 16, 0, 5, 0), (10, 8, 128, 16, 3, 0, 0), (10, 8, 128, 16, 3, 5, 3),
                (1 << 31, 8, 128, 16, 3, 5, 0), (10, 8, 128, 128, 3, 1 << 24, 0)):
        assert lib.ee_paged_cache_bytes(*bad) == 0, bad


def test_init_checks(pkg, lib):
    c = pkg.paged._PagedCacheC()
    shape = (8, 2, 128, 16, 2, 4, 0)
    need = lib.ee_paged_cache_bytes(*shape)
    assert lib.ee_paged_cache_init(None, 256, need, *shape, None) == INVALID
    assert lib.ee_paged_cache_init(ctypes.byref(c), 256, need - 1, *shape, None) == INVALID
    assert "too small" in pkg._lib.last_error()
    assert lib.ee_paged_cache_init(ctypes.byref(c), None, need, *shape, None) == INVALID
    assert lib.ee_paged_cache_init(ctypes.byref(c), 272, need, *shape, None) == MISALIGNED
    assert lib.ee_paged_cache_init(ctypes.byref(c), 256, need, 8, 2, 100, 16, 2, 4, 0, None) == INVALID


def _append(lib, cache, step, k=256, ldk=256, v=256, ldv=256, cos=256, sin=256, ldcs=128, q=256, ldq=512, heads=4,
            out=256, ldo=512):
    return lib.ee_paged_append(cache, step, k, ldk, v, ldv, cos, sin, ldcs, q, ldq, heads, out, ldo, None)


def test_append_checks(pkg, lib):
    c, s = _cache(pkg), _step(pkg)
    assert _append(lib, c, _step(pkg, rows=0)) == 0 and _append(lib, c, _step(pkg, batch=0)) == 0
    assert _append(lib, None, s) == INVALID and _append(lib, c, None) == INVALID
    assert _append(lib, _cache(pkg, table=None), s) == INVALID
    assert _append(lib, _cache(pkg, page_size=24), s) == INVALID
    assert _append(lib, _cache(pkg, tier=7), s) == INVALID
    assert _append(lib, _cache(pkg, scale=None), s) == INVALID
    assert _append(lib, _cache(pkg, pages=264), s) == MISALIGNED
    assert _append(lib, c, _step(pkg, rows=-1)) == INVALID and _append(lib, c, _step(pkg, cu=None)) == INVALID
    assert _append(lib, c, _step(pkg, rows=1 << 31)) == UNSUPPORTED
    assert _append(lib, c, s, k=None) == INVALID and _append(lib, c, s, v=None) == INVALID
    assert _append(lib, c, s, cos=None) == INVALID and "cos and sin" in pkg._lib.last_error()
    assert _append(lib, c, s, q=None) == INVALID and _append(lib, c, s, out=None) == INVALID
    assert _append(lib, c, s, k=264) == MISALIGNED and _append(lib, c, s, ldv=255) == MISALIGNED
    assert _append(lib, c, s, ldk=260) == MISALIGNED and _append(lib, c, s, ldcs=120) == MISALIGNED
    assert _append(lib, c, s, heads=0) == INVALID and _append(lib, c, s, ldq=504) == MISALIGNED
    assert _append(lib, c, _step(pkg, rows=(1 << 31) - 1), ldq=8192, ldo=8192, heads=64) == UNSUPPORTED


def test_read_checks(pkg, lib):
    c, s = _cache(pkg), _step(pkg)
    assert lib.ee_paged_read(c, _step(pkg, rows=0), None, 0, None, 0, None) == 0
    assert lib.ee_paged_read(c, s, None, 256, 256, 256, None) == INVALID
    assert lib.ee_paged_read(c, s, 256, 248, 256, 256, None) == MISALIGNED
    assert lib.ee_paged_read(None, s, 256, 256, 256, 256, None) == INVALID


def _attend(lib, cache, step, ws, q=256, ldq=512, heads=4, scale=0.1, out=256, ldo=512, H=256, wsp=256):
    return lib.ee_paged_attention(cache, step, q, ldq, heads, scale, out, ldo, H, wsp, ws, None)


def test_attention_checks(pkg, lib):
    c, s = _cache(pkg), _step(pkg)
    ws = lib.ee_paged_workspace_bytes(c)
    assert ws > lib.ee_paged_workspace_head_bytes() > 0
    assert lib.ee_paged_workspace_bytes(None) == 0
    assert _attend(lib, c, _step(pkg, rows=0), ws) == 0
    assert _attend(lib, c, s, ws, heads=3) == UNSUPPORTED and _attend(lib, c, s, ws, heads=0) == UNSUPPORTED
    assert _attend(lib, c, s, ws, scale=0.0) == INVALID and _attend(lib, c, s, ws, scale=float("nan")) == INVALID
    assert _attend(lib, c, s, ws, scale=float("inf")) == INVALID
    assert _attend(lib, c, s, ws, q=None) == INVALID and _attend(lib, c, s, ws, out=None) == INVALID
    assert _attend(lib, c, s, ws, q=260) == MISALIGNED and _attend(lib, c, s, ws, ldo=500) == MISALIGNED
    assert _attend(lib, c, s, ws, H=258) == MISALIGNED
    assert _attend(lib, c, s, ws - 1) == INVALID and _attend(lib, c, s, ws, wsp=None) == INVALID
    assert _attend(lib, c, s, ws, wsp=264) == MISALIGNED


class _HostCache:
    """PagedKVCache's host side alone."""

    def __new__(cls, pkg, **kw):
        import torch

        c = object.__new__(pkg.PagedKVCache)
        c.max_seqs, c.num_pages, c.page_size, c.max_pages = 3, 6, 16, 4
        c.tier, c.device = pkg.PrecisionTier.INT8, torch.device("cpu")
        c.table = torch.full((3, 4), -1, dtype=torch.int32)
        c.lengths, c._wide, c._pages = [0] * 3, [0] * 3, [[], [], []]
        c._free, c._changed = list(range(5, -1, -1)), {}
        return c


def test_pages_on_the_host(pkg):
    c = _HostCache(pkg)
    st = c.step([2, 0], counts=[33, 1])
    assert st.rows == 34 and st.c.max_new == 33
    assert st.arrays.tolist() == [2, 0, 0, 0, 33, 1, 0, 33, 34]
    assert c.table.tolist() == [[3, -1, -1, -1], [-1] * 4, [0, 1, 2, -1]] and c.free_pages == 2
    c.release(2)
    c.step([1], counts=[64])
    assert c.table[2].tolist() == [-1] * 4 and sorted(c.table[1].tolist()) == [0, 1, 2, 4]
    with pytest.raises(RuntimeError, match="full"):
        c.step([0], counts=[33])
    with pytest.raises(RuntimeError, match="more than 4 pages"):
        c.step([0], counts=[65])
    for bad in (dict(seqs=[3]), dict(seqs=[-1]), dict(seqs=[0, 0]), dict(seqs=[0], counts=[-1]),
                dict(seqs=[0], starts=[-2]), dict(seqs=[0], counts=[1, 2]), dict(seqs=[0], starts=[])):
        with pytest.raises(RuntimeError):
            c.step(**bad)
    with pytest.raises(RuntimeError, match="inside its sequence"):
        c.span([1], [0], [1])


def test_tensor_checks(pkg):
    import torch

    c = _HostCache(pkg)
    c.kv_heads, c.head_dim = 2, 64
    st = c.step([0], counts=[3])
    x = torch.zeros(3, 128, dtype=torch.float16)
    c.device, c._index = torch.device("cuda:0"), 0
    for call in (lambda: c.append(x, x, st), lambda: c.attention(x, st)):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()
    with pytest.raises(RuntimeError, match="multiple of kv_heads"):
        c.attention(torch.zeros(3, 192, dtype=torch.float16), st)
