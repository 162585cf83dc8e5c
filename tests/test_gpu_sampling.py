"""Softmax of logits and verification of drafted tokens on the GPU against plain numpy
in 64 bits (kv_ref)."""
import sys

import numpy as np
import pytest

import kv_ref as R
from conftest import bits

EPS = 2.0 ** -24


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def dev(a):
    from final_amd import hip
    return hip.DeviceArray.from_numpy(np.ascontiguousarray(a))


def run_softmax(dx, dy, rows, dim, t, **kw):
    from final_amd import hip, lfm
    need = lfm.softmax_workspace(rows, dim)
    ws = hip.DeviceArray((max(need, 16),), np.uint8)
    ws.fill_async(0xFF)
    lfm.softmax(dx, dy, rows, dim, temperature=t, workspace=ws, workspace_bytes=need, **kw)
    return dy.download()


def close(got, x, t):
    """A weight's exponent, at most |a| = (max - x) / t, takes three roundings (the difference, 1 / t, the
    product), so the weight is off by 3 |a| and 3 for exp itself.  It is the product (1) of a weight under
    its thread's maximum and that one's weight under the row's, whose |a| add up to it: 3 |a| + 7.  In the
    sum a third factor comes between, the wave's: 3 |a| + 11 on average over the weights, and log2(dim) + 80
    for its additions (threads sum at most 65 each); the quotient by 3.
    Below 2^-126 by two steps of the subnormal grid, or all of it."""
    ref = R.softmax(x, t)
    with np.errstate(invalid="ignore"):
        a = (x.astype(np.float64).max(1, keepdims=True) - x) / np.float64(np.float32(t))
    a = np.where(ref > 0, np.minimum(a, 800.0), 0.0)
    of_sum = (ref * (3 * a + 11)).sum(1, keepdims=True) + np.log2(x.shape[1] + 1) + 80
    tol = ref * EPS * (3 * a + 10 + of_sum) + 2.0 ** -126
    assert np.array_equal(np.isfinite(got), np.isfinite(ref))
    err = np.abs(got - ref)
    assert (err <= tol).all(), float((err / tol).max())
    assert np.all(got[ref == 0] <= 2.0 ** -126)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 2), (1, 65536), (2, 65537), (5, 1000), (1, 4099), (300, 4096),
                                      (17, 16385), (257, 8191), (1, 150001), (260, 65539), (64, 65536), (33, 65535),
                                      (32, 65532), (300, 40000), (401, 33000), (127, 32768), (128, 32769), (5, 9001)])
@pytest.mark.parametrize("t", [1.0, 0.3])
def test_softmax(rows, dim, t):
    say(f"[softmax] rows={rows} dim={dim} t={t}")
    r = np.random.default_rng(rows + dim)
    x = 3 * r.standard_normal((rows, dim), dtype=np.float32)
    x[0, dim // 2] = 40.0
    close(run_softmax(dev(x), dev(np.zeros_like(x)), rows, dim, t), x, t)


@pytest.mark.gpu
def test_softmax_of_more_rows_than_a_launch():
    rows, dim = (1 << 22) + 3, 2
    say(f"[softmax] rows={rows} dim={dim}")
    x = 3 * np.random.default_rng(22).standard_normal((rows, dim), dtype=np.float32)
    close(run_softmax(dev(x), dev(np.zeros_like(x)), rows, dim, 1.0), x, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dim", [(4, 700), (4, 65536), (300, 9001)])
def test_softmax_of_masks_and_extremes(rows, dim):
    r = np.random.default_rng(dim)
    x = r.standard_normal((rows, dim), dtype=np.float32)
    x[0, ::3] = -np.inf
    x[1] = -np.inf
    x[2, 5:] = np.finfo(np.float32).min  # the lowest value as a mask
    x[3] = np.finfo(np.float32).max
    x[3, 1] = -np.finfo(np.float32).max
    got = run_softmax(dev(x), dev(np.zeros_like(x)), rows, dim, 0.7)
    close(got, x, 0.7)
    assert not got[1].any() and not got[2, 5:].any() and got[3, 1] == 0
    x[0, 7], x[2, 0], x[3, 0] = np.nan, np.inf, -np.inf
    bad = run_softmax(dev(x), dev(np.zeros_like(x)), rows, dim, 0.7)
    assert np.isnan(bad[[0, 2]]).all() and np.isfinite(bad[3]).all() and not bad[1].any()
    if rows > 4:  # the other rows keep their bits
        assert np.array_equal(bits(bad[4:]), bits(got[4:]))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dim,xs,ys,shift", [(3, 1000, 1003, 1001, 1), (2, 65536, 65540, 65536, 0), (260, 513, 513, 520, 3)])
def test_softmax_strides_and_in_place(rows, dim, xs, ys, shift):
    from final_amd import hip
    r = np.random.default_rng(dim)
    flat = r.standard_normal(rows * xs + 8, dtype=np.float32)
    dx, out = dev(flat), np.full(rows * ys + 8, 7.0, np.float32)
    dy = dev(out)
    x = np.stack([flat[shift + i * xs:shift + i * xs + dim] for i in range(rows)])
    from final_amd import lfm
    need = lfm.softmax_workspace(rows, dim)
    ws = hip.DeviceArray((max(need, 16),), np.uint8)
    lfm.softmax(dx.ptr + 4 * shift, dy.ptr + 4 * shift, rows, dim, temperature=0.9, x_stride=xs, y_stride=ys, workspace=ws,
                workspace_bytes=need)
    got = dy.download()
    y = np.stack([got[shift + i * ys:shift + i * ys + dim] for i in range(rows)])
    close(y, x, 0.9)
    mask = np.ones(len(got), bool)
    for i in range(rows):
        mask[shift + i * ys:shift + i * ys + dim] = False
    assert (got[mask] == 7.0).all() and np.array_equal(bits(dx.download()), bits(flat))
    lfm.softmax(dx.ptr + 4 * shift, dx.ptr + 4 * shift, rows, dim, temperature=0.9, x_stride=xs, workspace=ws,
                y_stride=xs, workspace_bytes=need)
    got = dx.download()
    assert np.array_equal(bits(np.stack([got[shift + i * xs:shift + i * xs + dim] for i in range(rows)])), bits(y))


# -- verification ---------------------------------------------------------------

def probs(r, *shape, sharp=2.0):
    x = sharp * r.standard_normal(shape)
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def run_verify(t, d, ids, ua, us, n=None, vocab=None):
    from final_amd import hip, lfm
    B, K1, V = t.shape
    keep = [dev(a) if a is not None and a.size else None for a in (t, d, ids, ua, us, n)]
    acc, tok = dev(np.full(B, -9, np.int32)), dev(np.full((B, K1), -9, np.int32))
    need = lfm.verify_draft_workspace(B, V)
    ws = hip.DeviceArray((max(need, 16),), np.uint8)
    ws.fill_async(0xFF)
    lfm.verify_draft(keep[0], keep[1], keep[2], keep[3], keep[4], acc, tok, B, K1 - 1, V, n_valid=keep[5], workspace=ws,
                     workspace_bytes=need)
    return acc.download(), tok.download()


def same(got, want):
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]), (got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("B,K,V", [(1, 0, 1), (1, 4, 65536), (3, 1, 2), (7, 3, 1001), (64, 4, 4096), (2, 8, 65537),
                                   (5, 0, 150001), (300, 2, 700), (33, 16, 999), (3, 2, 8191), (3, 2, 8193), (2, 3, 16383),
                                   (2, 3, 16384), (2, 3, 16385), (4, 0, 16384), (2, 1024, 40), (1, 1024, 17000)])
def test_verify(B, K, V):
    say(f"[verify] B={B} K={K} V={V}")
    r = np.random.default_rng(B + K + V)
    t = probs(r, B, K + 1, V)
    d = (0.8 * t[:, :K] + 0.2 * probs(r, B, K, V)).astype(np.float32)
    ids = np.array([[R.draw(d[b, i].astype(np.float64), r.random()) for i in range(K)] for b in range(B)],
                   np.int32).reshape(B, K)
    ua, us = r.random((B, K), dtype=np.float32), r.random(B, dtype=np.float32)
    n = np.full(B, K, np.int32)
    want = R.verify(t, d, ids, ua, us, n)
    same(run_verify(t, d, ids, ua, us), want)
    n = r.integers(-2, K + 3, B).astype(np.int32)  # held to [0, K]
    same(run_verify(t, d, ids, ua, us, n), R.verify(t, d, ids, ua, us, n))
    if B == 64:
        assert 0 < want[0].mean() < K  # both outcomes were there


@pytest.mark.gpu
@pytest.mark.parametrize("V", [5, 1000, 10001, 16384, 65536, 70001])
def test_verify_borders(V):
    """Equal distributions, one-hot ones, zeros, random numbers at both ends, ids outside, NaN and negative weights."""
    r = np.random.default_rng(V)
    K = 2
    top = np.nextafter(np.float32(1), np.float32(0))
    t, d = probs(r, 12, K + 1, V), probs(r, 12, K, V)
    ids = r.integers(0, V, (12, K)).astype(np.int32)
    ua, us = np.full((12, K), 0.5, np.float32), np.array([0, top] * 6, np.float32)
    d[0] = t[0, :K]                      # equal: u < 1 accepts both
    d[1], ua[1] = t[1, :K], top
    t[2, 0], d[2, 0], ids[2, 0] = 0, 0, 1   # 0 < 0: rejected, nothing to draw from
    t[3, 0], t[3, 0, V - 1], ids[3, 0] = 0, 1, V - 1  # one-hot on the last id
    d[3, 0], t[3, 1], t[3, 1, V - 2], ids[3, 1] = 0.25 / V, 0, 1, 0
    ids[4, 0], ids[5, 0], ids[6, 1] = -1, V, 1 << 30
    t[7, 0, ::2], t[7, 0, 1] = np.nan, -3.0
    ids[7, 0] = 0
    t[8, 0], d[8, 0], ids[8, 0] = d[8, 0], t[8, 0], 3
    t[9, 0], d[9, 0] = t[9, 0] * np.float32(0.5), 1.0  # never above the draft: drawn from the target
    ids[9, 0], ua[9, 0] = 2, top
    t[10, 0, 4:], us[10] = 0, top
    ua[11], d[11, :, :] = 0, 0           # a draft of probability 0 under u = 0
    with np.errstate(invalid="ignore"):
        want = R.verify(t, d, ids, ua, us, np.full(12, K))
    assert want[0][0] == want[0][1] == 2 and want[1][2, 0] == -1 and want[0][3] == 1 and want[1][9, 0] >= 0
    same(run_verify(t, d, ids, ua, us), want)


@pytest.mark.gpu
def test_verify_of_strided_ids():
    from final_amd import hip, lfm
    r = np.random.default_rng(8)
    B, K, V = 5, 3, 900
    t, d = probs(r, B, K + 1, V), probs(r, B, K, V)
    rows = r.integers(0, V, (B, 11)).astype(np.int32)
    ua, us = 0.01 * r.random((B, K), dtype=np.float32), r.random(B, dtype=np.float32)
    ids = dev(rows)
    acc, tok = hip.DeviceArray((B,), np.int32), hip.DeviceArray((B, K + 1), np.int32)
    need = lfm.verify_draft_workspace(B, V)
    ws = hip.DeviceArray((need,), np.uint8)
    lfm.verify_draft(dev(t), dev(d), ids.ptr + 4 * 8, dev(ua), dev(us), acc, tok, B, K, V, ids_stride=11, workspace=ws,
                     workspace_bytes=need)
    want = R.verify(t, d, rows[:, 8:], ua, us, np.full(B, K))
    assert want[0].max() > 0
    same((acc.download(), tok.download()), want)


@pytest.mark.gpu
def test_model_verify():
    """The model's path: its probabilities are the softmax of the logits its head gives at each position,
    and its tokens what verification of them gives; n_draft = 0 draws the next token."""
    from final_amd import _native, hip, lfm
    r = np.random.default_rng(6)
    B, S, K, V, H, temp = 3, 20, 4, lfm.VOCAB, lfm.HIDDEN, 0.8
    model = lfm.LFM2Model(num_layers=2, layer_types=[1, 0], num_dense_layers=1, max_batch=4, max_seq=32, seed=5)
    ids = r.integers(0, V, (B, S)).astype(np.int32)
    dids = dev(ids)
    d = probs(r, B, K, V)
    d[0] = np.float32(1e-9)  # its drafts are accepted
    ua, us = r.random((B, K), dtype=np.float32), r.random(B, dtype=np.float32)
    n = np.array([K, K, 2], np.int32)
    pt, acc, tok = hip.DeviceArray((B, K + 1, V)), hip.DeviceArray((B,), np.int32), hip.DeviceArray((B, K + 1), np.int32)
    model.verify(dids, B, S, K, dev(d), dev(ua), dev(us), pt, acc, tok, temperature=temp, n_valid=dev(n))
    p = pt.download()
    same((acc.download(), tok.download()), R.verify(p, d, ids[:, S - K:], ua, us, n))
    assert acc.download()[0] == K
    # the head of shortened sequences of the same hidden states
    h = hip.DeviceArray((B * S, H))
    model.embed(dids, B, S, h)
    for layer in range(2):
        model.layer_forward(layer, h, B, S)
    hs = h.download().reshape(B, S, H)
    logits = hip.DeviceArray((B, V))
    for i in range(K + 1):
        m = S - K + i
        model.head(dev(hs[:, :m]), B, m, logits)
        x = logits.download()
        # the head's products of 2048 values round in another order there: 2048 + 6 steps of 2^-24 of the sum
        # of their magnitudes, which sqrt(2048) |h| |w| bounds; |h| is the norm's sqrt(2048), |w| below 1.1
        w = np.exp((2 * 2054 * EPS * np.sqrt(2048) * 1.1) / temp) - 1
        ref = R.softmax(x, temp)
        assert np.abs(p[:, i] - ref).max() <= (2 * w + 1e-5) * ref.max()
    assert model.status() == 0
    t0 = hip.DeviceArray((B, 1), np.int32)
    p0 = hip.DeviceArray((B, 1, V))
    model.verify(dids, B, S, 0, None, None, dev(us), p0, acc, t0, temperature=temp)
    same((acc.download(), t0.download()), R.verify(p0.download(), None, None, None, us, np.zeros(B)))
    for args in ((B, S, S), (B, S, -1), (5, S, K), (B, 33, K)):
        with pytest.raises(_native.MoeError) as e:
            model.verify(dids, *args, dev(d), dev(ua), dev(us), pt, acc, tok)
        assert e.value.status == _native.MOE_ERR_INVALID_ARG
    with pytest.raises(_native.MoeError) as e:
        model.verify(dids, B, S, K, dev(d), dev(ua), dev(us), pt, acc, tok, temperature=0.0)
    assert e.value.status == _native.MOE_ERR_INVALID_ARG
    model.close()


@pytest.mark.gpu
def test_model_verify_of_many_positions():
    """64 x 257 positions of 65536 logits are more than one product of the head takes: the last position's
    probabilities of every sequence are those of its forward."""
    import ctypes

    from final_amd import hip, lfm
    B, S, K, V, temp = 64, 260, 256, lfm.VOCAB, 1.0
    r = np.random.default_rng(7)
    model = lfm.LFM2Model(num_layers=1, layer_types=[1], num_dense_layers=1, max_batch=B, max_seq=S, seed=5)
    ids = r.integers(0, V, (B, S)).astype(np.int32)
    dids, logits = dev(ids), hip.DeviceArray((B, V))
    model.forward(dids, B, S, logits)
    ref = R.softmax(logits.download(), temp)
    p, d = hip.DeviceArray((B, K + 1, V)), hip.DeviceArray((B, K, V))
    d.fill_async(0)  # u * 0 < p: every draft is accepted
    ua, us = dev(r.random((B, K), dtype=np.float32)), r.random(B, dtype=np.float32)
    acc, tok = hip.DeviceArray((B,), np.int32), hip.DeviceArray((B, K + 1), np.int32)
    model.verify(dids, B, S, K, d, ua, dev(us), p, acc, tok, temperature=temp)
    assert (acc.download() == K).all()
    got = tok.download()
    assert np.array_equal(got[:, :K], ids[:, S - K:])
    row = np.empty((1, V), np.float32)
    w = np.exp((2 * 2054 * EPS * np.sqrt(2048) * 1.1) / temp) - 1  # as in test_model_verify
    for b in range(B):
        assert hip.rt().hipMemcpy(row.ctypes.data, p.ptr + 4 * ((b * (K + 1) + K) * V), row.nbytes, 2) == 0
        assert np.abs(row[0] - ref[b]).max() <= (2 * w + 1e-5) * ref[b].max()
        assert got[b, K] == R.verify(row[None], None, None, None, us[b:b + 1], np.zeros(1))[1][0, 0]
    model.close()


@pytest.mark.gpu
def test_model_verify_refuses_more_drafts_than_verification_takes():
    from final_amd import _native, hip, lfm
    model = lfm.LFM2Model(num_layers=1, layer_types=[1], num_dense_layers=1, max_batch=1, max_seq=1026, seed=5)
    x = hip.DeviceArray((16,))  # refused before anything reads it
    with pytest.raises(_native.MoeError) as e:
        model.verify(x, 1, 1026, 1025, x, x, x, x, x, x)
    assert e.value.status == _native.MOE_ERR_INVALID_ARG
    model.close()


@pytest.mark.gpu
def test_verify_of_many_random_numbers():
    """One distribution at many random numbers: every id is drawn at its place of the running sum."""
    r = np.random.default_rng(0)
    V, B = 3001, 2000
    p = probs(r, V)
    t = np.broadcast_to(p, (B, 1, V))
    us = np.sort(r.random(B, dtype=np.float32))
    got = run_verify(np.ascontiguousarray(t), None, None, None, us)
    want = R.verify(np.ascontiguousarray(t), None, None, None, us, np.zeros(B))
    same(got, want)


@pytest.mark.gpu
def test_logits_to_verified_tokens():
    """Head logits of drafts through softmax (in place) and verification, as a step with drafts runs them."""
    from final_amd import lfm
    r = np.random.default_rng(4)
    B, K, V = 6, 3, lfm.VOCAB
    logits = (2 * r.standard_normal((B * (K + 1), V))).astype(np.float32)
    dl = (logits.reshape(B, K + 1, V)[:, :K] + 0.5 * r.standard_normal((B, K, V))).astype(np.float32).reshape(B * K, V)
    t, d = dev(logits), dev(dl)
    pt = run_softmax(t, t, B * (K + 1), V, 0.8).reshape(B, K + 1, V)
    pd = run_softmax(d, d, B * K, V, 0.8).reshape(B, K, V)
    us = r.random(B, dtype=np.float32)
    # the drafts: one token each from the draft's probabilities, by the same operator
    ids = np.stack([run_verify(np.ascontiguousarray(pd[:, i:i + 1]), None, None, None, r.random(B, dtype=np.float32))[1][:, 0]
                    for i in range(K)], 1).astype(np.int32)
    assert (ids >= 0).all()
    ua = r.random((B, K), dtype=np.float32)
    same(run_verify(pt, pd, ids, ua, us), R.verify(pt, pd, ids, ua, us, np.full(B, K)))


@pytest.mark.gpu
def test_a_step_with_drafts_as_a_graph():
    """Keys and values written, attention, a head, softmax and verification, captured once and replayed with
    eager work between, as the sequences advance by what was accepted: each replay's bits are the eager ones."""
    import ctypes

    from final_amd import hip, lfm
    r = np.random.default_rng(8)
    B, K, V, page, per, prefix = 3, 2, 1024, 16, 12, 70
    N, front = K + 1, -(-prefix // page)
    pages = B * per + front
    cos, sin = lfm.rope_tables(prefix + per * page)
    weights = dev(r.standard_normal((V, 2048), dtype=np.float32) / 8)
    qw, kw, dc, ds = dev(np.ones(64, np.float32)), dev(np.ones(64, np.float32)), dev(cos), dev(sin)
    order = r.permutation(pages).astype(np.int32)
    table, shared = dev(order[:B * per].reshape(B, per)), dev(order[B * per:])
    start = r.standard_normal((2, pages, 8, page, 64)).astype(np.float16)
    own = np.array([K + 1, 30, 100], np.int32)

    class Side:
        def __init__(self):
            self.k, self.v = (dev(np.clip(a * 40, -127, 127).astype(np.int8)) for a in start)
            self.ks, self.vs = (dev(np.full((pages, 8, page), 0.02, np.float32)) for _ in range(2))
            self.c = lfm.KVCache(lfm.KV_INT8, pages, page, self.k, self.v, self.ks, self.vs)
            self.len = dev(own)
            self.b = lfm.KVBatch(B, self.len, table, per, max_new=N, max_len=128, prefix_pages=shared, prefix_len=prefix)
            self.x, self.o = hip.DeviceArray((B * N, lfm.QKV_COLS)), hip.DeviceArray((B * N, 2048))
            self.p, self.d = hip.DeviceArray((B * N, V)), hip.DeviceArray((B * K, V))
            self.ids, self.acc, self.tok = (hip.DeviceArray(n, np.int32) for n in ((B, K), (B,), (B, N)))
            self.ua, self.us = hip.DeviceArray((B, K)), hip.DeviceArray((B,))
            self.need = [lfm.kv_attention_workspace(self.c, self.b), lfm.softmax_workspace(B * N, V),
                         lfm.verify_draft_workspace(B, V)]
            self.ws = hip.DeviceArray((max(self.need),), np.uint8)  # the calls follow one another

        def step(self, st):
            lfm.kv_write(self.c, self.b, self.x, lfm.QKV_COLS, q_weight=qw, k_weight=kw, cos=dc, sin=ds, max_pos=len(cos),
                         stream=st)
            lfm.kv_attention(self.c, self.b, self.x, lfm.QKV_COLS, self.o, workspace=self.ws,
                             workspace_bytes=self.need[0], stream=st)
            lfm.gemm_nt(self.o, weights, self.p, B * N, V, 2048, stream=st)
            lfm.softmax(self.p, self.p, B * N, V, temperature=0.9, workspace=self.ws, workspace_bytes=self.need[1],
                        stream=st)
            lfm.verify_draft(self.p, self.d, self.ids, self.ua, self.us, self.acc, self.tok, B, K, V, workspace=self.ws,
                             workspace_bytes=self.need[2], stream=st)

    H, vp = hip.rt(), ctypes.c_void_p
    graphed, eager, st = Side(), Side(), hip.Stream()
    H.hipStreamBeginCapture.argtypes = [vp, ctypes.c_int]
    H.hipStreamEndCapture.argtypes = [vp, ctypes.POINTER(vp)]
    H.hipGraphInstantiate.argtypes = [ctypes.POINTER(vp), vp, vp, vp, ctypes.c_size_t]
    H.hipGraphLaunch.argtypes = [vp, vp]
    graph, ex = vp(), vp()
    assert H.hipStreamBeginCapture(st.handle, 2) == 0
    graphed.step(st)
    assert H.hipStreamEndCapture(st.handle, ctypes.byref(graph)) == 0
    assert H.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, 0) == 0
    for t in range(6):
        x = r.standard_normal((B * N, lfm.QKV_COLS), dtype=np.float32)
        ids, d = r.integers(0, V, (B, K)).astype(np.int32), np.full((B * K, V), 1.0 / V, np.float32)
        ua, us = r.random((B, K), dtype=np.float32), r.random(B, dtype=np.float32)
        for side in (graphed, eager):
            for a, b in ((side.x, x), (side.d, d), (side.ids, ids), (side.ua, ua), (side.us, us), (side.len, own)):
                a.upload(b)
        assert H.hipGraphLaunch(ex, st.handle) == 0
        st.synchronize()
        eager.step(None)
        hip.synchronize()
        for a, b in ((graphed.o, eager.o), (graphed.p, eager.p), (graphed.acc, eager.acc), (graphed.tok, eager.tok),
                     (graphed.k, eager.k), (graphed.vs, eager.vs)):
            a, b = a.download(), b.download()
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8)), t
        p = eager.p.download().reshape(B, N, V)
        want = R.verify(p, d.reshape(B, K, V), ids, ua, us, np.full(B, K))
        same((graphed.acc.download(), graphed.tok.download()), want)
        own += want[0].astype(np.int32) + 1
    H.hipGraphExecDestroy(ex)
    H.hipGraphDestroy(graph)
