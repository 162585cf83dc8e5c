"""Refusals of the cache, attention, softmax and verification entry points, which
answer before any GPU call; and the plain forms the GPU tests compare with."""
import ctypes

import numpy as np
import pytest

import kv_ref as R

A = 1 << 20  # an aligned address that no refused call looks at


@pytest.fixture(scope="module")
def lib():
    from final_amd import _native
    return _native


def cache(lib, **kw):
    d = dict(format=2, kv_heads=8, page_tokens=16, num_pages=4, k=A, v=A, k_scale=A, v_scale=A)
    d.update(kw)
    return lib.LfmKvCache(**d)


def batch(lib, **kw):
    d = dict(batch=2, tokens=4, max_new=2, max_len=10, new_start=None, own_len=A, pages=A, max_pages=3,
             prefix_pages=None, prefix_len=0)
    d.update(kw)
    return lib.LfmKvBatch(**d)


def write(lib, c, b, qkv=A, ld=48 * 64, heads=32, k_col=32 * 64, v_col=40 * 64, rope=(None,) * 4, max_pos=0):
    return lib.lib().lfm_kv_write(c and ctypes.byref(c), b and ctypes.byref(b), qkv, ld, heads, k_col, v_col, *rope,
                                  max_pos, None, None)


def read(lib, c, b, k=A, v=2 * A, rows=4, ld=512):
    return lib.lib().lfm_kv_read(ctypes.byref(c), ctypes.byref(b), k, v, rows, ld, None, None)


def attend(lib, c, b, q=A, ld=48 * 64, out=2 * A, ldo=32 * 64, heads=32, ws=A, n=1 << 40):
    return lib.lib().lfm_kv_attention(ctypes.byref(c), ctypes.byref(b), q, ld, out, ldo, heads, ws, n, None, None)


BAD_CACHES = [(dict(format=4), 2), (dict(format=-1), 2), (dict(kv_heads=0), 1), (dict(kv_heads=257), 2),
              (dict(page_tokens=8), 2), (dict(page_tokens=24), 2), (dict(page_tokens=8192), 2), (dict(page_tokens=0), 1),
              (dict(num_pages=0), 1), (dict(k=None), 1), (dict(v=A + 8), 1), (dict(k_scale=None), 1), (dict(v_scale=A + 4), 1),
              (dict(format=0), 1), (dict(format=1, k_scale=None), 1)]
BAD_BATCHES = [(dict(batch=-1), 1), (dict(tokens=5), 1), (dict(max_new=-1), 1), (dict(own_len=None), 1),
               (dict(pages=None), 1), (dict(prefix_len=1), 1), (dict(prefix_len=-1), 1), (dict(max_len=-1), 1),
               (dict(batch=65536, tokens=131072), 2), (dict(max_pages=1 << 27), 2), (dict(max_pages=-1), 1)]


@pytest.mark.parametrize("kw,want", BAD_CACHES)
def test_caches_refused(lib, kw, want):
    c, b = cache(lib, **kw), batch(lib)
    assert write(lib, c, b) == read(lib, c, b) == attend(lib, c, b) == want


@pytest.mark.parametrize("kw,want", BAD_BATCHES)
def test_batches_refused(lib, kw, want):
    c, b = cache(lib), batch(lib, **kw)
    assert write(lib, c, b) == read(lib, c, b) == attend(lib, c, b) == want


def test_arguments_refused(lib):
    c, b, L = cache(lib), batch(lib), lib.lib()
    inv, uns = lib.MOE_ERR_INVALID_ARG, lib.MOE_ERR_UNSUPPORTED
    assert write(lib, None, b) == inv and write(lib, c, None) == inv
    for kw in (dict(qkv=None), dict(qkv=A + 4), dict(ld=47 * 64), dict(ld=48 * 64 + 2), dict(k_col=2), dict(k_col=-4),
               dict(v_col=39 * 64), dict(rope=(A, A, A, None), max_pos=9), dict(rope=(A,) * 4, max_pos=0),
               dict(rope=(A,) * 4, max_pos=9, heads=33), dict(rope=(A, A + 4, A, A), max_pos=9)):
        assert write(lib, c, b, **kw) == inv, kw
    for kw in (dict(rows=-1), dict(ld=508), dict(ld=514), dict(k=A + 4), dict(k=2 * A)):
        assert read(lib, c, b, **kw) == inv, kw
    for kw in (dict(q=None), dict(out=None), dict(out=A), dict(ld=32 * 64 - 4), dict(ldo=32 * 64 - 4), dict(heads=0),
               dict(heads=12), dict(out=A + 8), dict(ldo=32 * 64 + 1)):
        assert attend(lib, c, b, **kw) == inv, kw
    assert attend(lib, c, b, heads=8 * 65, ld=8 * 65 * 64, ldo=8 * 65 * 64) == uns
    n = ctypes.c_size_t(7)
    big = batch(lib, max_len=4000, max_pages=250)
    assert L.lfm_kv_attention_workspace(ctypes.byref(c), ctypes.byref(big), 32, None) == inv
    assert L.lfm_kv_attention_workspace(ctypes.byref(c), ctypes.byref(big), 32, ctypes.byref(n)) == 0
    if n.value:
        assert attend(lib, c, big, ws=None) == inv and attend(lib, c, big, n=n.value - 1) == inv
        assert attend(lib, c, big, ws=A + 8) == inv
    # 2^24 blocks of 256 threads beside a prefix
    many = batch(lib, batch=65535, tokens=65535, max_new=1, prefix_len=16, prefix_pages=A)
    assert attend(lib, cache(lib, kv_heads=256), many, heads=256, ld=256 * 64, ldo=256 * 64, n=1 << 50) == uns
    # nothing to do
    for kw in (dict(batch=0, tokens=0), dict(max_new=0, tokens=0)):
        assert write(lib, c, batch(lib, **kw), qkv=None) == 0 and attend(lib, c, batch(lib, **kw), q=None) == 0
    assert read(lib, c, b, rows=0) == 0 and read(lib, c, b, k=None, v=None) == 0


def test_softmax_and_verify_refused(lib):
    L, inv = lib.lib(), lib.MOE_ERR_INVALID_ARG

    def soft(x=A, xs=10, y=2 * A, ys=10, rows=2, dim=10, t=1.0, ws=A, n=1 << 40):
        return L.lfm_softmax(x, xs, y, ys, rows, dim, t, ws, n, None)

    for kw in (dict(x=None), dict(y=None), dict(xs=9), dict(ys=9), dict(rows=-1), dict(dim=0), dict(t=0.0), dict(t=-1.0),
               dict(t=float("nan")), dict(t=float("inf")), dict(t=1e-40), dict(x=A, y=A, ys=11), dict(x=A + 2)):
        assert soft(**kw) == inv, kw
    assert soft(rows=0, x=None, y=None) == 0

    def ver(target=A, draft=A, ids=A, stride=3, ua=A, us=A, b=2, k=3, v=40000, acc=A, tok=A, ws=A, n=1 << 40):
        return L.lfm_verify_draft(target, draft, ids, stride, ua, us, None, b, k, v, acc, tok, ws, n, None)

    for kw in (dict(target=None), dict(draft=None), dict(ids=None), dict(ua=None), dict(us=None), dict(acc=None),
               dict(tok=None), dict(b=-1), dict(k=-1), dict(v=0), dict(stride=2), dict(ws=None), dict(n=1), dict(ws=A + 8)):
        assert ver(**kw) == inv, kw
    assert ver(k=1025) == ver(b=65536) == lib.MOE_ERR_UNSUPPORTED
    assert ver(b=0, target=None) == 0
    assert L.lfm_model_verify(None, A, 1, 4, 1, A, A, A, None, 1.0, A, A, A, None) == inv
    n = ctypes.c_size_t(0)
    assert L.lfm_softmax_workspace(-1, 4, ctypes.byref(n)) == L.lfm_softmax_workspace(1, 0, ctypes.byref(n)) == inv
    assert L.lfm_verify_draft_workspace(-1, 4, ctypes.byref(n)) == inv
    assert L.lfm_softmax_workspace(1, 70000, ctypes.byref(n)) == 0 and n.value > 0
    assert soft(rows=1, dim=70000, xs=70000, ys=70000, ws=None) == inv
    assert soft(rows=1, dim=70000, xs=70000, ys=70000, n=n.value - 1) == inv


def test_plain_forms():
    """The plain forms against values worked out by hand."""
    assert np.nanmax(R.E4M3) == 448 and R.E4M3[1] == 2.0 ** -9 and R.E4M3[8] == 2.0 ** -6
    y = np.array([17.0, 19.0, -17.0, 2.0 ** -10, 3 * 2.0 ** -10, 448.0])
    assert R.E4M3[R.to_e4m3(y)].tolist() == [16.0, 20.0, -16.0, 0.0, 2.0 ** -8, 448.0]
    assert R.to_bf16(np.array([1.00390625, 1.01171875], np.float32)).tolist() == [0x3F80, 0x3F82]
    x = np.zeros((3, 64), np.float32)
    x[0, :4] = [127.0, 0.5, 1.5, -2.5]
    x[1, 0] = np.inf
    q, s = R.store(x, R.INT8)
    assert s[0] == 1 and q[0, :4].tolist() == [127, 0, 2, -2] and np.isnan(s[1]) and s[2] == 0 and not q[2].any()
    o, _, _ = R.attention(np.zeros((2, 64)), np.ones((2, 64)), np.eye(2, 64), np.array([[1, 1], [0, 0]], bool))
    assert o[0, :2].tolist() == [0.5, 0.5] and not o[1].any()
    assert R.draw(np.array([0.0, 0.25, 0.75]), 0.0) == 1 and R.draw(np.array([0.0, 0.25, 0.75]), 0.25) == 2
    assert R.draw(np.zeros(3), 0.5) == -1
    assert R.softmax(np.array([[0.0, -np.inf], [-np.inf, -np.inf]], np.float32), 1.0).tolist() == [[1, 0], [0, 0]]
