"""The paged KV cache on the GPU against plain numpy (kv_ref): rows written and read
back bit for bit, attention over pages and a shared prefix within bounds counted from
its roundings, and what the contract says of contents that do not fit."""
import sys

import numpy as np
import pytest

import kv_ref as R
from conftest import bits

FMTS = [R.F32, R.BF16, R.INT8, R.FP8]
EPS = 2.0 ** -24


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def dev(a):
    from final_amd import hip
    return hip.DeviceArray.from_numpy(np.ascontiguousarray(a))


class Pool:
    """A cache whose every byte is set (`fill`), on the device and as numpy arrays."""

    def __init__(self, fmt, kv, page, pages, fill=0xFF):
        from final_amd import lfm
        self.fmt, self.kv, self.page, self.pages = fmt, kv, page, pages
        shape = (pages, kv, page, 64)
        self.data = [np.full(shape, 0, R.DTYPE[fmt]) for _ in range(2)]
        self.scale = [np.zeros(shape[:3], np.float32) for _ in range(2)]
        for a in self.data + self.scale:
            a.view(np.uint8)[...] = fill
        scaled = fmt in (R.INT8, R.FP8)
        self.d = [dev(a) for a in self.data]
        self.s = [dev(a) for a in self.scale] if scaled else [None, None]
        self.c = lfm.KVCache(fmt, pages, page, self.d[0], self.d[1], self.s[0], self.s[1], kv_heads=kv)

    def put(self, table, pos, rows):
        """Writes rows [2][n][kv][64] fp32 at positions `pos` of a page table into the numpy side."""
        pg, off = np.asarray(table)[pos // self.page], pos % self.page
        for i in range(2):
            q, s = R.store(rows[i], self.fmt)
            self.data[i][pg, :, off] = q
            if s is not None:
                self.scale[i][pg, :, off] = s

    def upload(self):
        for i in range(2):
            self.d[i].upload(self.data[i])
            if self.s[i] is not None:
                self.s[i].upload(self.scale[i])

    def get(self, table, n):
        """fp32 values [2][n][kv][64] of positions 0 .. n of a page table, numpy side."""
        pos = np.arange(n)
        pg, off = np.asarray(table)[pos // self.page], pos % self.page
        return [R.values(self.data[i][pg, :, off], self.scale[i][pg, :, off], self.fmt) for i in range(2)]

    def same(self):
        """The device holds what the numpy side does, byte for byte (NaN scales by being NaN)."""
        for i in range(2):
            got = self.d[i].download()
            off = np.argwhere(got.view(np.uint8) != self.data[i].view(np.uint8))
            assert not len(off), ("kv"[i], len(off), off[0].tolist(), got[tuple(off[0][:3])], self.data[i][tuple(off[0][:3])])
            if self.s[i] is not None:
                a, b = self.s[i].download(), self.scale[i]
                assert np.array_equal(np.isnan(a), np.isnan(b))
                assert np.array_equal(bits(a)[~np.isnan(b)], bits(b)[~np.isnan(b)])


class Seqs:
    """Sequences with `n` new tokens and own lengths `own`, on pages of a random order."""

    def __init__(self, r, pool, n, own, prefix=0, uniform=False, max_pages=None, max_len=None):
        from final_amd import lfm
        B = len(n)
        self.n, self.own, self.prefix = np.array(n), np.array(own, np.int32), prefix
        self.per = max_pages or max(1, -(-int(max(own)) // pool.page))
        front = -(-prefix // pool.page)
        order = r.permutation(pool.pages)[:B * self.per + front].astype(np.int32)
        assert len(order) == B * self.per + front
        self.table, self.front = order[:B * self.per].reshape(B, self.per), order[B * self.per:]
        self.start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        self.tokens = int(self.start[-1])
        self.d = [dev(self.own), dev(self.table), dev(self.front if front else np.zeros(1, np.int32)), dev(self.start)]
        self.c = lfm.KVBatch(B, self.d[0], self.d[1], self.per, max_new=int(max(n)), max_len=max_len or int(max(own)),
                             tokens=self.tokens, new_start=None if uniform else self.d[3],
                             prefix_pages=self.d[2] if front else None, prefix_len=prefix)

    def new_pos(self, b):
        return np.arange(self.own[b] - self.n[b], self.own[b])

    def rows(self, b):
        return slice(self.start[b], self.start[b + 1])


def draws(r, shape, sizes=True):
    """Normal rows, of magnitudes from 2^-20 to 2^20 where `sizes`."""
    x = r.standard_normal(shape, dtype=np.float32)
    if sizes:
        x = np.ldexp(x, r.integers(-20, 21, shape[:-1])[..., None]).astype(np.float32)
    return x


SHAPES = [  # kv heads, page, new, own, uniform
    (8, 16, [1], [37], True), (8, 32, [1, 1, 1], [1, 33, 64], True), (8, 16, [5, 1, 7, 0], [5, 16, 40, 3], False),
    (2, 128, [130, 17], [130, 400], False), (1, 16, [16, 16], [16, 48], True), (3, 64, [9], [200], False)]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("kv,page,new,own,uniform", SHAPES)
def test_write_and_read(fmt, kv, page, new, own, uniform):
    from final_amd import hip, lfm
    say(f"[kv] fmt={fmt} kv={kv} page={page} new={new} own={own}")
    r = np.random.default_rng(fmt + 10 * kv)
    pool = Pool(fmt, kv, page, len(new) * -(-max(own) // page) + 3)
    q = Seqs(r, pool, new, own, uniform=uniform)
    heads, pad = 4 * kv, 8  # unused columns between and behind the blocks
    k_col, v_col = heads * 64 + pad, heads * 64 + kv * 64 + 2 * pad
    ld = v_col + kv * 64 + pad
    x = draws(r, (q.tokens, ld // 4, 4)).reshape(q.tokens, ld)
    k = x[:, k_col:k_col + kv * 64].reshape(-1, kv, 64)
    k[0, 0] = 0.0                             # a row of zeros
    k[-1, -1, 5] = np.inf
    v = x[:, v_col:v_col + kv * 64].reshape(-1, kv, 64)
    v[-1, 0, 9] = np.nan
    v[0, -1] = np.float32(2.0 ** -140)        # subnormal, equal
    x[:, k_col:k_col + kv * 64], x[:, v_col:v_col + kv * 64] = k.reshape(-1, kv * 64), v.reshape(-1, kv * 64)
    dx, flag = dev(x), dev(np.zeros(1, np.int32))
    lfm.kv_write(pool.c, q.c, dx, ld, heads=heads, k_col=k_col, v_col=v_col, bad_flag=flag)
    for b in range(len(new)):
        pool.put(q.table[b], q.new_pos(b), [k[q.rows(b)], v[q.rows(b)]])
    pool.same()
    assert np.array_equal(bits(dx.download()), bits(x)) and flag.download()[0] == 0
    # back, into rows with room to spare and into fewer than there are
    for rows in (max(own) + 3, max(1, max(own) - 5)):
        ldo = kv * 64 + 4
        out = [np.full((len(new) * rows, ldo), 7.0, np.float32) for _ in range(2)]
        d = [dev(o) for o in out]
        lfm.kv_read(pool.c, q.c, d[0], d[1], rows, ld=ldo, bad_flag=flag)
        for b in range(len(new)):
            m = min(own[b], rows)
            for i, val in enumerate(pool.get(q.table[b], m)):
                out[i][b * rows:b * rows + m, :kv * 64] = val.reshape(m, kv * 64)
        for i in range(2):
            got = d[i].download()
            assert np.array_equal(got, out[i], equal_nan=True)
        one = dev(np.zeros_like(out[1]))
        lfm.kv_read(pool.c, q.c, None, one, rows, ld=ldo)
        sel = out[1].copy()
        sel[:, kv * 64:] = 0
        got = one.download()
        for b in range(len(new)):
            m = min(own[b], rows)
            assert np.array_equal(got[b * rows:b * rows + m], sel[b * rows:b * rows + m], equal_nan=True)
            assert not got[b * rows + m:(b + 1) * rows].any()
    assert flag.download()[0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [R.INT8, R.FP8, R.BF16])
def test_rounding_borders(fmt):
    """Halves, values beside them, the largest and the smallest magnitudes."""
    from final_amd import lfm
    r = np.random.default_rng(3)
    kv, page, T = 8, 16, 64
    pool = Pool(fmt, kv, page, T // page)
    q = Seqs(r, pool, [T], [T])
    x = np.zeros((T, 2, kv, 64), np.float32)
    rows = x.reshape(-1, 64)
    top = {R.INT8: 127.0, R.FP8: 448.0, R.BF16: 1.0}[fmt]
    for i in range(len(rows)):
        steps = r.integers(0, 126, 64) + 0.5 if fmt == R.INT8 else r.integers(8, 16, 64) * 2.0 ** r.integers(-9, 4, 64) + \
            2.0 ** r.integers(-10, 3, 64)
        z = (steps * r.choice([-1, 1], 64)).astype(np.float32)
        z = np.nextafter(z, np.float32(r.choice([-1e9, 1e9])), dtype=np.float32) if i % 3 == 1 else z
        z = np.clip(z, -top, top)
        z[i % 64] = top
        s = [1.0, 2.0 ** -126, 2.0 ** 100, 2.0 ** -140, 1.7, 1e-38, 7e35 if fmt == R.FP8 else 2e36, 3.0][(i // 3) % 8]
        with np.errstate(over="ignore"):
            rows[i] = np.clip((z.astype(np.float64) * s), -3.3e38, 3.3e38).astype(np.float32)
    h = np.ascontiguousarray(x.reshape(T, -1))
    lfm.kv_write(pool.c, q.c, dev(h), h.shape[1], k_col=0, v_col=kv * 64)
    pool.put(q.table[0], np.arange(T), [x[:, 0], x[:, 1]])
    pool.same()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads,kv,new,own,prefix", [(32, 8, [1, 1], [1, 70], 0), (32, 8, [40, 3], [40, 90], 21),
                                                     (6, 3, [2], [50], 7)])
def test_write_with_norm_and_rotation(fmt, heads, kv, new, own, prefix):
    """q in place and k in the cache are lfm_qk_norm_rope's, bit for bit."""
    from final_amd import lfm
    r = np.random.default_rng(heads + len(new))
    pool = Pool(fmt, kv, 16, len(new) * -(-max(own) // 16) + 1 + -(-prefix // 16))
    q = Seqs(r, pool, new, own, prefix=prefix)
    ld, k_col, v_col = (heads + 2 * kv) * 64, heads * 64, (heads + kv) * 64
    x = draws(r, (q.tokens, ld), sizes=False)
    qw, kw = (dev(1 + 0.1 * r.standard_normal(64, dtype=np.float32)) for _ in range(2))
    cos, sin = lfm.rope_tables(prefix + max(own))
    dc, ds = dev(cos), dev(sin)
    ref = np.empty_like(x)
    for b in range(len(new)):  # a sequence's rows stand next to each other, and so do their positions
        d = dev(x[q.rows(b)])
        at = (prefix + own[b] - new[b]) * 256
        lfm.qk_norm_rope(d, ld, qw, kw, dc.ptr + at, ds.ptr + at, 1, new[b], heads=heads, kv_heads=kv, k_col=k_col)
        ref[q.rows(b)] = d.download()
    dx, flag = dev(x), dev(np.zeros(1, np.int32))
    lfm.kv_write(pool.c, q.c, dx, ld, heads=heads, k_col=k_col, v_col=v_col, q_weight=qw, k_weight=kw, cos=dc, sin=ds,
                 max_pos=len(cos), bad_flag=flag)
    for b in range(len(new)):
        t = ref[q.rows(b)]
        pool.put(q.table[b], q.new_pos(b), [t[:, k_col:v_col].reshape(-1, kv, 64), t[:, v_col:].reshape(-1, kv, 64)])
    pool.same()
    assert np.array_equal(bits(dx.download()[:, :k_col]), bits(ref[:, :k_col])) and flag.download()[0] == 0
    assert np.array_equal(bits(dx.download()[:, k_col:]), bits(x[:, k_col:]))
    # a table one position short leaves the last position's tokens out
    last = int(np.argmax(own))
    before = [d.download() for d in pool.d]
    dx.upload(x)
    lfm.kv_write(pool.c, q.c, dx, ld, heads=heads, k_col=k_col, v_col=v_col, q_weight=qw, k_weight=kw, cos=dc, sin=ds,
                 max_pos=len(cos) - 1, bad_flag=flag)
    assert flag.download()[0] == 1
    assert all(np.array_equal(a.view(np.uint8), d.download().view(np.uint8)) for a, d in zip(before, pool.d))
    t = q.start[last + 1] - 1
    assert np.array_equal(bits(dx.download()[t]), bits(x[t]))


def attend(pool, q, x, heads, out=None, flag=None, stream=None, ws=None):
    from final_amd import hip, lfm
    dx = x if isinstance(x, hip.DeviceArray) else dev(x)
    do = out or dev(np.full((q.tokens, heads * 64), 7.0, np.float32))
    need = lfm.kv_attention_workspace(pool.c, q.c, heads=heads)
    ws = ws or hip.DeviceArray((max(need, 16),), np.uint8)
    ws.fill_async(0xFF, stream)
    lfm.kv_attention(pool.c, q.c, dx, dx.shape[1], do, heads=heads, workspace=ws, workspace_bytes=need, bad_flag=flag,
                     stream=stream)
    if stream:
        stream.synchronize()
    return do.download()


def fill(r, pool, q, sizes=False):
    """Every position of the prefix and of the sequences, in numpy and on the device."""
    def rows(n):
        return [draws(r, (n, pool.kv, 64), sizes) for _ in range(2)]
    if q.prefix:
        pool.put(q.front, np.arange(q.prefix), rows(q.prefix))
    for b in range(len(q.own)):
        pool.put(q.table[b], np.arange(q.own[b]), rows(q.own[b]))
    pool.upload()


def check(pool, q, x, heads, got, hide=None, skip=()):
    """Against 64 bits.  With a key's score off by d, its weight is off by a factor e^(2 d)
    (numerator and sum), so an output by 2 d sum p|v|.  d: q's scaling and at most 64 sums
    round (66 steps of sum |q||k| / 8), and exp's argument, no larger than twice that plus
    the scores' spread, rounds twice.  Then N sums of p v, of p, a weight's and an output's
    few roundings: N + 24 steps.  fp32 has no weights below 2^-126 of the largest (they may
    count as 0), nor products of a weight with a row's scale (a stored value is at most 448):
    N 2^-126 max(|v|, 448) off at most, where the sum of weights is at least 1."""
    G = heads // pool.kv
    fk, fv = pool.get(q.front, q.prefix) if q.prefix else (np.zeros((0, pool.kv, 64), np.float32),) * 2
    worst = 0.0
    for b in range(len(q.own)):
        if b in skip:
            continue
        k, v = pool.get(q.table[b], q.own[b])
        k, v = np.concatenate([fk, k]), np.concatenate([fv, v])
        i = np.arange(q.n[b])
        vis = np.arange(len(k))[None] <= (q.prefix + q.own[b] - q.n[b] + i)[:, None]
        if hide is not None:
            vis = vis & ~hide(b, len(k))[None]
        for h in range(heads):
            qr = x[q.rows(b), h * 64:(h + 1) * 64]
            ref, mag, size = R.attention(qr, k[:, h // G], v[:, h // G], vis)
            d = (66 + 4) * EPS * size + 4 * EPS
            tol = (2 * d[:, None] + (len(k) + 24) * EPS) * mag + len(k) * 2.0 ** -126 * max(448.0, np.abs(v[:, h // G]).max())
            err = np.abs(got[q.rows(b), h * 64:(h + 1) * 64] - ref)
            assert (err <= tol).all(), (b, h, float((err / tol).max()))
            worst = max(worst, float((err / np.maximum(tol, 1e-300)).max(initial=0.0)))
    say(f"  worst error: {worst:.3f} of the bound")


CASES = [  # heads, kv, page, new, own, prefix
    (32, 8, 16, [1], [1], 0), (32, 8, 16, [1], [300], 0), (32, 8, 32, [1, 1, 1, 1], [31, 32, 33, 65], 0),
    (32, 8, 16, [1, 1, 1], [7, 150, 16], 129), (32, 8, 64, [5, 3, 0, 8], [5, 200, 9, 64], 33),
    (8, 8, 16, [1, 2], [40, 1000], 0), (16, 2, 32, [4, 1], [100, 2], 64), (64, 1, 16, [2], [77], 48),
    (6, 3, 128, [33], [33], 0), (32, 8, 128, [100, 37], [300, 37], 500), (5, 5, 16, [17, 16], [17, 90], 15),
    (32, 8, 16, [1] * 70, list(range(1, 71)), 40), (12, 1, 16, [1], [4000], 0),
    # one to four column tiles of own positions, alone, beside a prefix of one column tile and of several
    (32, 8, 16, [3], [100], 70), (32, 8, 32, [3, 2], [100, 600], 300), (32, 8, 16, [6, 2], [9, 700], 0),
    (32, 8, 16, [4], [600], 0), (16, 8, 64, [1, 2, 1], [600, 2, 31], 1500), (64, 8, 16, [2], [40], 2100),
    # prefixes long enough to be shared, where those above are read by each sequence
    (32, 8, 16, [1, 1, 1], [7, 150, 16], 2129), (32, 8, 64, [5, 3, 0, 8], [5, 200, 9, 64], 1633),
    (5, 5, 16, [17, 16], [17, 90], 1515), (16, 2, 32, [4, 1], [100, 2], 2064), (64, 1, 16, [2], [77], 648),
    (32, 8, 32, [1], [1], 2048), (32, 8, 16, [1] * 70, list(range(1, 71)), 1200),
    # two blocks on a CU, with a prefix and without
    (32, 8, 16, [3] * 40, list(range(3, 43)), 40), (32, 8, 16, [2, 3] * 20, list(range(3, 43)), 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads,kv,page,new,own,prefix", CASES)
def test_attention(fmt, heads, kv, page, new, own, prefix):
    say(f"[kv attention] fmt={fmt} heads={heads}/{kv} page={page} new={new[:4]} own={own[:4]} prefix={prefix}")
    r = np.random.default_rng(fmt + heads + len(new))
    pool = Pool(fmt, kv, page, len(new) * -(-max(own) // page) + -(-prefix // page) + 2)  # bytes of NaN where unwritten
    q = Seqs(r, pool, new, own, prefix=prefix, uniform=len(set(new)) == 1)
    fill(r, pool, q)
    x = 2 * draws(r, (q.tokens, heads * 64 + 20), sizes=False)
    flag = dev(np.zeros(1, np.int32))
    got = attend(pool, q, x, heads, flag=flag)
    assert np.isfinite(got).all() and flag.download()[0] == 0
    check(pool, q, x, heads, got)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [R.BF16, R.FP8])
@pytest.mark.parametrize("heads,kv,page,new,own,prefix,max_len", [
    (4, 1, 16, [1], [9000], 0, 1),            # one part: more than 32 tiles a wave
    (4, 1, 32, [1, 1], [9000, 40], 0, 1 << 20),  # a hint far above the lengths
    (32, 8, 64, [512], [512], 4200, 512)])    # and of the prefix
def test_attention_of_many_tiles_a_wave(fmt, heads, kv, page, new, own, prefix, max_len):
    say(f"[kv attention] fmt={fmt} heads={heads}/{kv} new={new} own={own} prefix={prefix} hint={max_len}")
    r = np.random.default_rng(fmt)
    pool = Pool(fmt, kv, page, len(new) * -(-max(own) // page) + -(-prefix // page) + 2)
    q = Seqs(r, pool, new, own, prefix=prefix, max_len=max_len)
    fill(r, pool, q)
    x = draws(r, (q.tokens, heads * 64), sizes=False)
    got = attend(pool, q, x, heads)
    check(pool, q, x, heads, got)
    assert np.array_equal(bits(attend(pool, q, x, heads)), bits(got))  # and the same bits again


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,new,longest", [(R.F32, 1, 992), (R.INT8, 1, 2016), (R.BF16, 3, 2016), (R.F32, 3, 992),
                                             (R.INT8, 5, 1504), (R.F32, 5, 736), (R.FP8, 9, 736)])
def test_attention_around_the_length_that_is_split(fmt, new, longest):
    r = np.random.default_rng(longest)
    pool = Pool(fmt, 8, 32, 140)
    for own in (longest, longest + 1):
        say(f"[kv attention] fmt={fmt} new={new} own={own}")
        q = Seqs(r, pool, [new, new], [own, longest // 2])
        fill(r, pool, q)
        x = draws(r, (q.tokens, 2048), sizes=False)
        check(pool, q, x, 32, attend(pool, q, x, 32))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_pages_listed_more_than_once(fmt):
    """Sequences that share pages with each other, with the prefix and with themselves."""
    r = np.random.default_rng(fmt)
    pool = Pool(fmt, 8, 16, 40)
    q = Seqs(r, pool, [2, 1, 1], [90, 70, 33], prefix=40)
    q.table[1, :4] = q.table[0, :4]  # positions 0 .. 63 alike
    q.table[2, :2] = q.front[0]      # the prefix's first page, twice
    q.d[1].upload(q.table)
    fill(r, pool, q)
    x = draws(r, (q.tokens, 2048), sizes=False)
    check(pool, q, x, 32, attend(pool, q, x, 32))


@pytest.mark.gpu
def test_output_rows_of_their_own_length():
    from final_amd import hip, lfm
    r = np.random.default_rng(4)
    pool = Pool(R.INT8, 8, 16, 60)
    q = Seqs(r, pool, [2, 1], [300, 35], prefix=100)
    fill(r, pool, q)
    x = draws(r, (q.tokens, 2048), sizes=False)
    want = attend(pool, q, x, 32)
    wide = np.zeros((q.tokens, 2048 + 12), np.float32)
    wide[:, 8:8 + 2048] = x
    dx, do = dev(wide), dev(np.full((q.tokens, 2052), 7.0, np.float32))
    need = lfm.kv_attention_workspace(pool.c, q.c)
    ws = hip.DeviceArray((max(need, 16),), np.uint8)
    lfm.kv_attention(pool.c, q.c, dx.ptr + 32, 2060, do, ld_out=2052, workspace=ws, workspace_bytes=need)
    got = do.download()
    assert np.array_equal(bits(got[:, :2048]), bits(want)) and (got[:, 2048:] == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [R.INT8, R.F32])
def test_pages_beyond_4_gib(fmt):
    """The same sequence in a pool's first and last pages, whose addresses are 4.5 GB and more apart."""
    from final_amd import hip, lfm
    r = np.random.default_rng(fmt)
    size = np.dtype(R.DTYPE[fmt]).itemsize
    page_bytes = 8 * 4096 * 64 * size
    pages = (9 << 29) // page_bytes
    k, v = (hip.DeviceArray((pages * page_bytes,), np.uint8) for _ in range(2))
    scaled = fmt == R.INT8
    ks, vs = ((hip.DeviceArray((pages * 8 * 4096,)) for _ in range(2)) if scaled else (None, None))
    cache = lfm.KVCache(fmt, pages, 4096, k, v, ks, vs)
    n = 5000
    x = dev(draws(r, (n, lfm.QKV_COLS), sizes=False))
    own, got = dev(np.array([n], np.int32)), []
    for table in ([0, 1], [pages - 1, pages - 2]):
        t = dev(np.array([table], np.int32))
        b = lfm.KVBatch(1, own, t, 2, max_new=n, max_len=n)
        flag = dev(np.zeros(1, np.int32))
        lfm.kv_write(cache, b, x, lfm.QKV_COLS, bad_flag=flag)
        out = [hip.DeviceArray((n, 512)) for _ in range(2)]
        lfm.kv_read(cache, b, out[0], out[1], n, bad_flag=flag)
        one = lfm.KVBatch(1, own, t, 2, max_new=1, max_len=n)
        need = lfm.kv_attention_workspace(cache, one)
        ws, o = hip.DeviceArray((max(need, 16),), np.uint8), hip.DeviceArray((1, 2048))
        lfm.kv_attention(cache, one, x, lfm.QKV_COLS, o, workspace=ws, workspace_bytes=need, bad_flag=flag)
        got.append([a.download() for a in out + [o]])
        assert flag.download()[0] == 0
    assert all(np.array_equal(bits(a), bits(b)) for a, b in zip(*got))
    if fmt == R.F32:
        assert np.array_equal(bits(got[0][0]), bits(x.download()[:, 2048:2560]))


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [100, 2100])  # read by each sequence, and shared
@pytest.mark.parametrize("fmt", FMTS)
def test_attention_of_large_scores(fmt, prefix):
    """Scores of a few hundred, of either sign, values of magnitudes 2^-20 to 2^20."""
    r = np.random.default_rng(fmt)
    pool = Pool(fmt, 8, 16, 190)
    q = Seqs(r, pool, [3, 1], [90, 200], prefix=prefix)
    fill(r, pool, q, sizes=True)
    x = np.ldexp(draws(r, (q.tokens, 2048), sizes=False), -14).astype(np.float32)
    check(pool, q, x, 32, attend(pool, q, x, 32))
    x[:, :64] = 0.0  # equal weights
    x[:, 64:128] = -np.abs(x[:, 64:128]) * 2.0 ** 100  # far below any sentinel
    got = attend(pool, q, x, 32)
    assert np.isfinite(got[:, :64]).all() and not np.isnan(got).any()


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [40, 2090])
@pytest.mark.parametrize("fmt", FMTS)
def test_attention_does_not_see_the_future(fmt, prefix):
    """What stands behind a token's own position, not finite ones included, changes none of its bits."""
    r = np.random.default_rng(fmt)
    pool = Pool(fmt, 8, 16, 170)
    q = Seqs(r, pool, [4, 3], [50, 35], prefix=prefix)
    fill(r, pool, q)
    x = draws(r, (q.tokens, 2048), sizes=False)
    clean = attend(pool, q, x, 32)
    for val in (np.nan, np.inf, -np.inf):
        for which in range(2):
            rows = [np.ones((1, 8, 64), np.float32) for _ in range(2)]
            rows[which][...] = val
            for b in range(2):
                pool.put(q.table[b], np.array([q.own[b] - 1]), rows)
            pool.upload()
            got = attend(pool, q, x, 32)
            last = [3, 6]
            keep = [0, 1, 2, 4, 5]
            assert np.array_equal(bits(got[keep]), bits(clean[keep]))
            assert not np.isfinite(got[last]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("prefix,at", [(40, 3), (40, 39), (2090, 3), (2090, 2089)])
def test_not_finite_rows_reach_who_sees_them(fmt, prefix, at):
    """A row of the prefix reaches every token; one of a kv head's keys or values only its heads."""
    r = np.random.default_rng(fmt)
    pool = Pool(fmt, 8, 16, 170)
    q = Seqs(r, pool, [4, 1], [50, 35], prefix=prefix)
    fill(r, pool, q)
    x = draws(r, (q.tokens, 2048), sizes=False)
    clean = attend(pool, q, x, 32)
    for which in range(2):
        for val in (np.nan, np.inf):
            rows = [np.ones((1, 8, 64), np.float32) for _ in range(2)]
            rows[which][:, 3] = val
            saved = [a.copy() for a in pool.data + pool.scale]
            pg, off = q.front[at // 16], at % 16
            for i in range(2):
                d, sc = R.store(rows[i], fmt)
                pool.data[i][pg, 3, off] = d[0, 3]
                if sc is not None:
                    pool.scale[i][pg, 3, off] = sc[0, 3]
            pool.upload()
            got = attend(pool, q, x, 32).reshape(-1, 32, 64)
            assert not np.isfinite(got[:, 12:16]).any()
            keep = np.r_[0:12, 16:32]
            assert np.array_equal(bits(got[:, keep]), bits(clean.reshape(-1, 32, 64)[:, keep]))
            for a, b in zip(pool.data + pool.scale, saved):
                a[...] = b
            pool.upload()


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [40, 2090])
def test_attention_of_not_finite_queries(prefix):
    r = np.random.default_rng(1)
    pool = Pool(R.INT8, 8, 16, 170)
    q = Seqs(r, pool, [2, 2], [50, 35], prefix=prefix)
    fill(r, pool, q)
    x = draws(r, (q.tokens, 2048), sizes=False)
    clean = attend(pool, q, x, 32)
    x[1, 64 * 5 + 3], x[2, 64 * 31] = np.nan, np.inf
    got = attend(pool, q, x, 32)
    hit = np.zeros(got.shape, bool)
    hit[1, 64 * 5:64 * 6] = hit[2, 64 * 31:] = True
    assert np.isnan(got[hit]).all() and np.array_equal(bits(got[~hit]), bits(clean[~hit]))


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [40, 2088])
@pytest.mark.parametrize("fmt", FMTS)
def test_pages_outside_the_cache(fmt, prefix):
    from final_amd import hip, lfm
    r = np.random.default_rng(fmt)
    pool = Pool(fmt, 8, 16, 160)
    q = Seqs(r, pool, [2, 1, 1], [70, 35, 16], prefix=prefix)
    fill(r, pool, q)
    x = draws(r, (q.tokens, lfm.QKV_COLS), sizes=False)
    table, front = q.table.copy(), q.front.copy()
    table[0, 1], table[1, 2], table[2, 0], front[1] = pool.pages, -1, 1 << 30, -(1 << 31)
    q.d[1].upload(table)
    q.d[2].upload(front)

    def hide(b, n):
        j = np.arange(n) // 16
        own = (np.arange(n) - prefix) // 16
        return np.where(np.arange(n) < prefix, j == 1, own == [1, 2, 0][b])

    flag = dev(np.zeros(1, np.int32))
    got = attend(pool, q, x, 32, flag=flag)
    assert flag.download()[0] == 1
    check(pool, q, x, 32, got, hide=hide)
    # nothing to see at all
    front[:] = pool.pages + 69
    q.d[2].upload(front)
    assert not attend(pool, q, x, 32, flag=flag)[3].any()
    # reading back: zeros; writing: nothing
    flag.upload(np.zeros(1, np.int32))
    d = [hip.DeviceArray((3 * 70, 512)) for _ in range(2)]
    lfm.kv_read(pool.c, q.c, d[0], d[1], 70, bad_flag=flag)
    for got, val in zip((a.download().reshape(3, 70, 512) for a in d), pool.get(q.table[0], 70)):
        val = val.reshape(70, 512).copy()
        val[16:32] = 0
        assert np.array_equal(got[0], val) and not got[2, :16].any()
    assert flag.download()[0] == 1
    flag.upload(np.zeros(1, np.int32))
    lfm.kv_write(pool.c, q.c, dev(x), x.shape[1], bad_flag=flag, k_col=2048, v_col=2560)
    pool.put(q.table[0], q.new_pos(0), [x[:2, c:c + 512].reshape(2, 8, 64) for c in (2048, 2560)])
    pool.same()
    assert flag.download()[0] == 1


@pytest.mark.gpu
def test_sequences_that_do_not_fit():
    """Left out and flagged; own_len 0 left out without a flag; the others' results as without them."""
    from final_amd import lfm
    r = np.random.default_rng(5)
    pool = Pool(R.INT8, 8, 16, 40)
    q = Seqs(r, pool, [2, 2, 2, 2], [30, 40, 33, 20], max_pages=3)
    fill(r, pool, q)
    x = draws(r, (q.tokens, lfm.QKV_COLS), sizes=False)
    clean = attend(pool, q, x, 32)
    good = np.array([0, 1, 4, 5])
    bad = [(0, None, 0), (49, None, 1), (-1, None, 1), (1, None, 1), (1 << 31, None, 1), (40, [0, 2, 1, 6, 8], 1),
           (40, [0, 2, -4, 6, 8], 1), (40, [0, 2, 4, 6, 1 << 30], 1)]
    for own1, start, flagged in bad:
        own = q.own.astype(np.int64).copy()
        own[1] = own1
        q.d[0].upload(own.astype(np.uint32).view(np.int32))
        q.d[3].upload(np.array(start if start else q.start, np.int32))
        flag = dev(np.zeros(1, np.int32))
        got = attend(pool, q, x, 32, flag=flag)
        assert flag.download()[0] == flagged, (own1, start)
        left = [6, 7] if start and start[4] > 8 else [2, 3]
        if start and start[2] < 2:  # sequence 2's rows begin elsewhere as well
            assert np.array_equal(bits(got[[0, 1, 6, 7]]), bits(clean[[0, 1, 6, 7]]))
        else:
            keep = good if left == [2, 3] else np.arange(4)
            assert np.array_equal(bits(got[keep]), bits(clean[keep])) and (got[left] == 7.0).all()
        flag.upload(np.zeros(1, np.int32))
        if start is None:
            lfm.kv_write(pool.c, q.c, dev(x), x.shape[1], bad_flag=flag)
            assert flag.download()[0] == flagged
            out = dev(np.full((4 * 40, 512), 7.0, np.float32))
            lfm.kv_read(pool.c, q.c, out, None, 40, bad_flag=flag)
            if own1 != 1:
                assert (out.download().reshape(4, 40, 512)[1] == 7.0).all()
            pool.upload()


@pytest.mark.gpu
@pytest.mark.parametrize("batch,seq", [(2, 100), (3, 33)])
def test_steps_give_what_whole_sequences_give(batch, seq):
    """Prompts written and attended as chunks, then token by token, against lfm_attention on whole
    sequences, and behind a shared prefix against the same tokens as each sequence's own."""
    from final_amd import hip, lfm
    r = np.random.default_rng(seq)
    ld = lfm.QKV_COLS
    front = 40  # the first tokens of every sequence are the same
    x = draws(r, (batch, seq, ld), sizes=False)
    x[:, :front] = x[0, :front]
    front = min(front, seq - 3)
    qw, kw = (dev(1 + 0.1 * r.standard_normal(64, dtype=np.float32)) for _ in range(2))
    cos, sin = (dev(a) for a in lfm.rope_tables(seq))
    whole = dev(x.reshape(batch * seq, ld))
    lfm.qk_norm_rope(whole, ld, qw, kw, cos, sin, batch, seq)
    out = hip.DeviceArray((batch * seq, lfm.Q_COLS))
    lfm.attention(whole, ld, out, batch, seq)
    want = out.download().reshape(batch, seq, -1)
    qkv = whole.download().reshape(batch, seq, ld)
    # both sides round as test_attention counts
    q, k, v = qkv[..., :2048].reshape(batch, seq, 32, 64), qkv[..., 2048:2560], qkv[..., 2560:]
    size = np.abs(q.astype(np.float64)).sum(-1).max() * np.abs(k).max() / 8
    tol = 2 * (2 * (70 * EPS * size + 4 * EPS) + (seq + 24) * EPS) * np.abs(v).max()

    def step(pool, pages, b_own, n, prefix, prefix_pages, rows):
        B, per = pages.shape
        keep = [dev(np.full(B, b_own, np.int32)), dev(pages), dev(rows.reshape(B * n, ld)),
                dev(prefix_pages) if prefix else None, hip.DeviceArray((B * n, 2048))]
        c = lfm.KVBatch(B, keep[0], keep[1], per, max_new=n, max_len=b_own, prefix_pages=keep[3], prefix_len=prefix)
        lfm.kv_write(pool.c, c, keep[2], ld, q_weight=qw, k_weight=kw, cos=cos, sin=sin, max_pos=seq)
        need = lfm.kv_attention_workspace(pool.c, c)
        ws = hip.DeviceArray((max(need, 16),), np.uint8)
        lfm.kv_attention(pool.c, c, keep[2], ld, keep[4], workspace=ws, workspace_bytes=need)
        return keep[4].download().reshape(B, n, 2048)

    per = -(-seq // 16)
    for shared in (False, True):
        pool = Pool(R.F32, 8, 16, batch * per + per)
        order = r.permutation(pool.pages).astype(np.int32)
        pages, fp = order[:batch * per].reshape(batch, per), order[batch * per:]
        pre = front if shared else 0
        if shared:  # the prefix is written as a sequence of its own
            got = step(pool, fp[None], front, front, 0, None, x[:1, :front])
            assert np.abs(got[0] - want[0, :front]).max() <= tol
        at = 0
        chunk = (seq - pre) // 2
        while pre + at < seq:
            n = chunk if at == 0 else 1
            got = step(pool, pages, at + n, n, pre, fp, np.ascontiguousarray(x[:, pre + at:pre + at + n]))
            assert np.abs(got - want[:, pre + at:pre + at + n]).max() <= tol
            at += n


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [100, 2100])
def test_graph_replays_follow_the_lengths(prefix):
    """write + attention captured once, replayed as sequences grow, with eager work between."""
    import ctypes

    from final_amd import hip, lfm
    r = np.random.default_rng(9)
    H, vp = hip.rt(), ctypes.c_void_p
    pool, other = (Pool(R.FP8, 8, 16, 160) for _ in range(2))
    q = Seqs(r, pool, [1, 1, 1], [20, 3, 40], prefix=prefix, uniform=True, max_pages=8, max_len=64)
    fill(r, pool, q)
    for i in range(2):
        other.data[i][...], other.scale[i][...] = pool.data[i], pool.scale[i]
    other.upload()
    st = hip.Stream()
    x = dev(np.zeros((3, lfm.QKV_COLS), np.float32))
    out = hip.DeviceArray((3, 2048))
    need = lfm.kv_attention_workspace(pool.c, q.c)
    ws = hip.DeviceArray((max(need, 16),), np.uint8)
    H.hipStreamBeginCapture.argtypes = [vp, ctypes.c_int]
    H.hipStreamEndCapture.argtypes = [vp, ctypes.POINTER(vp)]
    H.hipGraphInstantiate.argtypes = [ctypes.POINTER(vp), vp, vp, vp, ctypes.c_size_t]
    H.hipGraphLaunch.argtypes = [vp, vp]
    graph, ex = vp(), vp()
    assert H.hipStreamBeginCapture(st.handle, 2) == 0
    lfm.kv_write(pool.c, q.c, x, lfm.QKV_COLS, stream=st)
    lfm.kv_attention(pool.c, q.c, x, lfm.QKV_COLS, out, workspace=ws, workspace_bytes=need, stream=st)
    assert H.hipStreamEndCapture(st.handle, ctypes.byref(graph)) == 0
    assert H.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, 0) == 0
    own = q.own.copy()
    for t in range(5):
        rows = draws(r, (3, lfm.QKV_COLS), sizes=False)
        x.upload(rows)
        q.d[0].upload(own)
        assert H.hipGraphLaunch(ex, st.handle) == 0
        st.synchronize()
        got = out.download()
        dx = dev(rows)
        lfm.kv_write(other.c, q.c, dx, lfm.QKV_COLS)
        eager = attend(other, q, dx, 32)
        assert np.array_equal(bits(got), bits(eager)), t
        assert np.array_equal(pool.d[0].download(), other.d[0].download())
        own += np.array([1, 3, 0], np.int32) if t % 2 else np.array([1, 1, 1], np.int32)
    H.hipGraphExecDestroy(ex)
    H.hipGraphDestroy(graph)


@pytest.mark.gpu
def test_two_streams():
    """Two calls at once on two streams, each with its own workspace, give what they give alone."""
    from final_amd import hip, lfm
    r = np.random.default_rng(2)
    pool = Pool(R.INT8, 8, 16, 200)
    qs = [Seqs(r, pool, [1] * 4, [300, 20, 250, 33], prefix=0, uniform=True), None]
    fill(r, pool, qs[0])
    qs[1] = qs[0]
    xs = [draws(r, (4, 2048), sizes=False) for _ in range(2)]
    alone = [attend(pool, q, x, 32) for q, x in zip(qs, xs)]
    st = [hip.Stream(), hip.Stream()]
    dx, out = [dev(x) for x in xs], [hip.DeviceArray((4, 2048)) for _ in xs]
    need = lfm.kv_attention_workspace(pool.c, qs[0].c)
    ws = [hip.DeviceArray((max(need, 16),), np.uint8) for _ in xs]
    hip.synchronize()
    for _ in range(8):
        for i in range(2):
            lfm.kv_attention(pool.c, qs[i].c, dx[i], 2048, out[i], workspace=ws[i], workspace_bytes=need, stream=st[i])
    for i in range(2):
        st[i].synchronize()
        assert np.array_equal(bits(out[i].download()), bits(alone[i]))
