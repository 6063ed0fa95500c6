"""The paged cache on the GPU: kv_append (norms, rotation, append over 16 and 4
bits), kv_read and attn_paged against the formulas in 64 bits, at the sizes,
masks, pages and lengths where they can go wrong."""
import numpy as np
import pytest

import _oracle as O
from _paged_ref import DT_BF16, DT_F16, Paged, near

pytestmark = pytest.mark.gpu

KEEP = 0x5A                                         # outputs start as this byte: what is left alone stays so


def say(*a):
    print(*a, flush=True)


def up(hip, a):
    return hip.Buffer.from_numpy(np.ascontiguousarray(a))


def kept(hip, nbytes):
    return up(hip, np.full(nbytes, KEEP, np.uint8))


def index_args(hip, P):
    return [up(hip, P.table), up(hip, P.len)] + ([up(hip, P.rows)] if P.ragged else [])


def append(hip, P, x, kpool, vpool, rope=0, norm=None, eps=1e-6, cos=None, sin=None, ldx=None):
    q, kb, vb = kept(hip, P.n * P.H * P.hd * 2 + 256), up(hip, kpool), up(hip, vpool)
    args = [q, kb, vb, up(hip, x)] + index_args(hip, P)
    args += [up(hip, g) for g in norm] if norm is not None else []
    args += [up(hip, cos), up(hip, sin)] if rope else []
    kw = P.spec(h=P.H, rope=rope, norm=int(norm is not None), eps=float(np.float32(eps)))
    if ldx:
        kw["ldx"] = ldx
    hip.builtin("kv_append", args, outs=(0, 1, 2), **kw)
    raw = q.read(np.uint8)
    assert (raw[P.n * P.H * P.hd * 2:] == KEEP).all()
    return raw[:P.n * P.H * P.hd * 2].view(np.uint16).reshape(P.n, P.H, P.hd), \
        kb.read(np.uint8).reshape(kpool.shape), vb.read(np.uint8).reshape(vpool.shape)


def attn(hip, P, q, kpool, vpool, scale, **kw):
    out = kept(hip, P.n * P.H * P.hd * 2 + 256)
    kw = P.spec(h=P.H, scale=float(scale), **kw)
    ws = kept(hip, hip.attn_paged_ws(**kw))
    hip.builtin("attn_paged", [out, up(hip, q), up(hip, kpool), up(hip, vpool)] + index_args(hip, P) + [ws], **kw)
    raw = out.read(np.uint8)
    assert (raw[P.n * P.H * P.hd * 2:] == KEEP).all()
    return raw[:P.n * P.H * P.hd * 2].view(np.uint16).reshape(P.n, P.H, P.hd)


def check_append(P, x, kpool, vpool, got, **kw):
    """Every row's q within f32's error and one rounding, k and v as the
    operator's own steps give them bit for bit, nothing else changed."""
    q, k1, v1 = got
    kw64 = dict(kw)
    wk, wv, owned = kpool.copy(), vpool.copy(), np.zeros(P.n, bool)
    for row, s, pos in P.each_row():
        owned[row] = True
        qq, _, _, eq, _ = P.project(x, row, pos, np.float64, **kw64)
        if not 0 <= pos < P.maxpages * P.page:
            assert (q[row] == 0).all(), row
        else:
            assert near(O.decode(q[row], P.dt).astype(np.float64), qq, eq, P.dt), row
        _, k, v, _, _ = P.project(x, row, pos, np.float32, **kw)
        at = P.where(s, pos)
        if at:
            P.put(wk, *at, k)
            P.put(wv, *at, v)
    assert np.array_equal(v1, wv)
    assert np.array_equal(k1, wk)
    assert (q[~owned].view(np.uint8) == KEEP).all()


def check_attn(P, q, kpool, vpool, got, scale):
    owned = np.zeros(P.n, bool)
    g = O.decode(got, P.dt).astype(np.float64)
    kheld, vheld = P.held(kpool), P.held(vpool)
    for row, s, pos in P.each_row():
        owned[row] = True
        want, tol = P.attend(q, kheld, vheld, row, s, pos, scale)
        assert near(g[row], want, tol, P.dt), (row, s, pos)
    assert (got[~owned].view(np.uint8) == KEEP).all()


SEQS = {"one": [(1, 1)], "one-17": [(1, 17)], "b3": [(1, 5), (1, 64), (1, 33)], "rows": [(7, 20)],
        "ragged": [(3, 40), (0, 12), (1, 1), (17, 17), (2, 130)], "empty": [(1, 0), (1, 3)]}


@pytest.mark.parametrize("dt", [DT_BF16, DT_F16])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("rope,norm", [(0, False), (1, False), (2, True), (1, True), (0, True)])
@pytest.mark.parametrize("H,Hkv,hd,page", [(4, 2, 64, 16), (8, 2, 128, 32), (5, 5, 64, 64), (3, 1, 128, 16)])
@pytest.mark.parametrize("seqs", SEQS)
def test_kv_append(hip, dt, bits, rope, norm, H, Hkv, hd, page, seqs):
    say(f"case: kv_append dt={dt} bits={bits} rope={rope} norm={norm} H={H} Hkv={Hkv} hd={hd} page={page} {seqs}")
    P = Paged(SEQS[seqs], dt, bits, H, Hkv, hd, page, extra=2 if seqs == "ragged" else 0)
    x, kpool, vpool = P.make_x(), P.stale(), P.filled()
    kw = dict(rope=rope)
    if norm:
        kw.update(norm=[(1 + 0.1 * P.rng.standard_normal(hd)).astype(np.float32) for _ in range(2)], eps=1e-5)
    if rope:
        kw["cos"], kw["sin"] = P.tables()
    check_append(P, x, kpool, vpool, append(hip, P, x, kpool, vpool, **kw), **kw)


@pytest.mark.parametrize("bits", [16, 4])
def test_kv_append_strides_holes_and_values(hip, bits):
    """Rows of x further apart than they are long, pages that are none, positions
    past the table, groups of zeros, huge, tiny, infinite and NaN values."""
    say(f"case: kv_append strides and values, bits={bits}")
    for dt in (DT_BF16, DT_F16):
        P = Paged([(5, 21), (4, 60), (3, 2)], dt, bits, 4, 2, 64, 16, holes=((0, 1, -1), (1, 2, 10 ** 6), (1, 3, -7)))
        P.len[1] = 81                               # the table's 5 pages end at 80
        P.seqs = [(5, 21), (4, 81), (3, 2)]
        ldx = 8 * 64 + 24
        x = P.make_x(ldx)
        v = O.decode(x, dt).reshape(x.shape)
        big = 3e38 if dt == DT_BF16 else 65504.0
        v[1, 6 * 64:7 * 64] = 0.0                   # a v head of zeros, then of extremes
        v[2, 6 * 64:6 * 64 + 32] = big
        v[2, 6 * 64 + 40] = big * 0.7
        v[3, 6 * 64:7 * 64] = 2.0 ** -24 if dt == DT_F16 else 1e-38
        v[5, 4 * 64 + 3] = np.inf                   # in k
        v[8, 7 * 64 + 60] = np.nan
        v[9, 6 * 64] = -np.inf
        x = O.encode(v.astype(np.float32), dt)
        kpool, vpool = P.filled(), P.stale()
        check_append(P, x, kpool, vpool, append(hip, P, x, kpool, vpool, ldx=ldx))


def test_kv_append_every_code_border(hip):
    """Values at and beside each border between two codes, in each place of a
    group; ties go to the even code."""
    say("case: kv_append code borders")
    P = Paged([(8, 8)], DT_F16, 4, 1, 1, 64, 16)
    b = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    t = np.concatenate([b, b * (1 + 2.0 ** -10), b * (1 - 2.0 ** -11), [6.0, 4.5, 5.9]])
    v = np.zeros((8, 3 * 64), np.float32)
    for r in range(8):
        for g in range(6):
            w = np.resize(np.roll(t, 5 * r + g), 32) * np.where(np.arange(32) % 3 == 1, -1, 1)
            w[(r + g) % 32] = 6.0
            v[r, 32 * g:32 * g + 32] = w * 2.0 ** (r - 4)
    x = O.encode(v, DT_F16)
    pool = P.stale()
    check_append(P, x, pool, pool, append(hip, P, x, pool, pool))


@pytest.mark.parametrize("dt,bits,H,Hkv,hd,page", [(DT_BF16, 16, 4, 2, 64, 16), (DT_F16, 4, 8, 8, 128, 32),
                                                   (DT_BF16, 4, 2, 1, 64, 64), (DT_F16, 16, 6, 3, 128, 16)])
def test_kv_read(hip, dt, bits, H, Hkv, hd, page):
    say(f"case: kv_read dt={dt} bits={bits} Hkv={Hkv} hd={hd} page={page}")
    seqs = [(40, 40), (3, 90), (0, 5), (2, 1), (1, 33)]
    P = Paged(seqs, dt, bits, H, Hkv, hd, page, extra=3, holes=((1, 88 // page, -1),))
    kpool, vpool = P.filled(), P.filled()
    nb = P.n * Hkv * hd * 2
    k, v = kept(hip, nb + 64), kept(hip, nb + 64)
    hip.builtin("kv_read", [k, v, up(hip, kpool), up(hip, vpool)] + index_args(hip, P), outs=(0, 1), **P.spec())
    owned = np.zeros(P.n, bool)
    k, v = k.read(np.uint8), v.read(np.uint8)
    assert (k[nb:] == KEEP).all() and (v[nb:] == KEEP).all()
    k, v = (z[:nb].view(np.uint16).reshape(P.n, Hkv, hd) for z in (k, v))
    for row, s, pos in P.each_row():
        owned[row] = True
        at = P.where(s, pos)
        for got, pool in ((k, kpool), (v, vpool)):
            want = P.get(pool, *at) if at else np.zeros((Hkv, hd))
            assert np.array_equal(O.decode(got[row], dt).astype(np.float64), want), (row, s, pos)
    assert (k[~owned].view(np.uint8) == KEEP).all() and (v[~owned].view(np.uint8) == KEEP).all()


ATTN = {"one": [(1, 1)], "one-16": [(1, 16)], "one-300": [(1, 300)], "b4": [(1, 63), (1, 64), (1, 65), (1, 0)],
        "verify": [(4, 4), (4, 70), (4, 129)], "rows-33": [(33, 33)], "chunk": [(20, 150)],
        "ragged": [(1, 200), (0, 12), (40, 40), (2, 130), (1, 1), (5, 17)],
        "many": [(1, 7 * i % 90 + 1) for i in range(70)], "negative": [(5, 3), (5, 9)]}


@pytest.mark.parametrize("dt", [DT_BF16, DT_F16])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("H,Hkv,hd,page", [(4, 1, 128, 16), (4, 2, 64, 32), (5, 5, 64, 16), (6, 2, 128, 64),
                                           (8, 1, 64, 16), (20, 1, 128, 32), (16, 2, 128, 128)])
@pytest.mark.parametrize("seqs", ATTN)
def test_attn_paged(hip, dt, bits, H, Hkv, hd, page, seqs):
    say(f"case: attn_paged dt={dt} bits={bits} H={H} Hkv={Hkv} hd={hd} page={page} {seqs}")
    P = Paged(ATTN[seqs], dt, bits, H, Hkv, hd, page, extra=3 if seqs == "ragged" else 0)
    q = O.encode((1.5 * P.rng.standard_normal((P.n, H, hd))).astype(np.float32), dt)
    kpool, vpool = P.filled(), P.filled()
    scale = np.float32(hd ** -0.5)
    kw = {} if seqs == "many" else dict(t=max(r for r, _ in P.seqs))
    check_attn(P, q, kpool, vpool, attn(hip, P, q, kpool, vpool, scale, **kw), scale)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("seqs", [[(1, 1500)], [(3, 2500), (3, 700)], [(130, 1000), (1, 900), (64, 64)]])
def test_attn_paged_long(hip, bits, seqs):
    """Contexts that the work is split over, and a prompt's rows beside single ones."""
    say(f"case: attn_paged long bits={bits} {seqs}")
    P = Paged(seqs, DT_BF16, bits, 8, 2, 128, 64)
    q = O.encode((1.5 * P.rng.standard_normal((P.n, 8, 128))).astype(np.float32), DT_BF16)
    kpool, vpool = P.filled(), P.filled()
    scale = np.float32(128 ** -0.5)
    check_attn(P, q, kpool, vpool, attn(hip, P, q, kpool, vpool, scale), scale)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("seqs", [[(1, 100), (1, 40)], [(4, 100), (4, 40)], [(50, 100), (1, 40)]])
def test_attn_paged_holes_and_capacity(hip, bits, seqs):
    """Rows whose page is none are not seen (a row with only such rows is zeros);
    a length past the table sees the table's rows."""
    say(f"case: attn_paged holes bits={bits} {seqs}")
    P = Paged(seqs, DT_F16, bits, 4, 2, 64, 16, holes=((0, 0, -1), (0, 2, 999), (0, 3, -5), (1, 0, -1), (1, 1, -1), (1, 2, -1)))
    P.len[0] = 400
    P.seqs = [(P.seqs[0][0], 400), P.seqs[1]]
    q = O.encode(P.rng.standard_normal((P.n, 4, 64)).astype(np.float32), DT_F16)
    kpool, vpool = P.filled(), P.filled()
    got = attn(hip, P, q, kpool, vpool, 0.125)
    check_attn(P, q, kpool, vpool, got, 0.125)
    assert (got[P.rows[1]:] == 0).all()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("seqs", [[(4, 60)], [(3, 17), (3, 16)], [(40, 75)], [(150, 150)]])
def test_attn_paged_later_positions_that_are_not_finite(hip, bits, bad, seqs):
    """K and V of one position hold NaN or infinities: earlier rows do not see
    them, its own and later ones do (a NaN key makes the whole row NaN; infinite
    values alone come through as they are)."""
    say(f"case: attn_paged not finite bits={bits} bad={bad} {seqs}")
    P = Paged(seqs, DT_BF16, bits, 4, 1, 128, 16)
    q = O.encode(P.rng.standard_normal((P.n, 4, 128)).astype(np.float32), DT_BF16)
    kpool, vpool = P.filled(), P.filled()
    s, pos = 0, seqs[0][1] - 2
    v = P.get(vpool, *P.where(s, pos))
    v[:, 5] = bad
    v[:, 100] = -bad
    P.put(vpool, *P.where(s, pos), v)
    got = attn(hip, P, q, kpool, vpool, 0.09)
    check_attn(P, q, kpool, vpool, got, 0.09)
    k = P.get(kpool, *P.where(s, pos))
    k[:, 7] = np.nan
    P.put(kpool, *P.where(s, pos), k)
    got = O.decode(attn(hip, P, q, kpool, vpool, 0.09), DT_BF16)
    kheld, vheld = P.held(kpool), P.held(vpool)
    for row, sq, p in P.each_row():
        if sq == s and p >= pos:
            assert np.isnan(got[row]).all(), row
        else:
            want, tol = P.attend(q, kheld, vheld, row, sq, p, 0.09)
            assert near(got[row].astype(np.float64), want, tol, DT_BF16), row


@pytest.mark.parametrize("scale", [0.0, -0.125, 3.0, 1e-38, -2e4])
@pytest.mark.parametrize("seqs", [[(1, 50), (1, 9)], [(40, 75), (33, 33)]])
def test_attn_paged_scales(hip, scale, seqs):
    """Any finite scale: none (the mean of the rows), negative, and so large that one row takes all."""
    say(f"case: attn_paged scale={scale} {seqs}")
    P = Paged(seqs, DT_BF16, 16, 4, 2, 64, 16)
    q = O.encode((0.01 * P.rng.standard_normal((P.n, 4, 64)) if abs(scale) > 10 else
                  P.rng.standard_normal((P.n, 4, 64))).astype(np.float32), DT_BF16)
    kpool, vpool = P.filled(), P.filled()
    scale = np.float32(scale)
    check_attn(P, q, kpool, vpool, attn(hip, P, q, kpool, vpool, scale), scale)


def test_attn_paged_t_leaves_longer_sequences_out(hip):
    say("case: attn_paged t")
    P = Paged([(1, 40), (6, 40), (2, 9)], DT_BF16, 16, 4, 2, 64, 16)
    q = O.encode(P.rng.standard_normal((P.n, 4, 64)).astype(np.float32), DT_BF16)
    kpool, vpool = P.filled(), P.filled()
    got = attn(hip, P, q, kpool, vpool, 0.125, t=2)
    assert (got[1:7].view(np.uint8) == KEEP).all()
    g = O.decode(got, DT_BF16).astype(np.float64)
    for row, s, pos in P.each_row():
        if s != 1:
            want, tol = P.attend(q, P.held(kpool), P.held(vpool), row, s, pos, 0.125)
            assert near(g[row], want, tol, DT_BF16), row


def test_paged_garbage_indexes_stay_inside(hip):
    """rows, len and table full of garbage: nothing outside the buffers is
    touched, the call ends, and a good call after it is right."""
    say("case: garbage rows, len and table")
    rng = np.random.default_rng(3)
    P = Paged([(3, 30), (2, 20), (9, 40)], DT_BF16, 16, 4, 2, 64, 16)
    q = O.encode(rng.standard_normal((P.n, 4, 64)).astype(np.float32), DT_BF16)
    x, kpool, vpool = P.make_x(), P.filled(), P.filled()
    good = attn(hip, P, q, kpool, vpool, 0.125)
    rows, ln, table = P.rows.copy(), P.len.copy(), P.table.copy()
    for i in range(6):
        P.rows = rng.integers(-2 ** 31, 2 ** 31, rows.shape).astype(np.int32) if i % 2 else rng.permutation(rows)
        P.len = rng.integers(-2 ** 31, 2 ** 31, ln.shape).astype(np.int32) if i % 3 else ln
        P.table = rng.integers(-2 ** 31, 2 ** 31, table.shape).astype(np.int32) if i % 4 > 1 else table
        append(hip, P, x, kpool, vpool)
        attn(hip, P, q, kpool, vpool, 0.125)
        nb = P.n * 2 * 64 * 2
        k, v = kept(hip, nb), kept(hip, nb)
        hip.builtin("kv_read", [k, v, up(hip, kpool), up(hip, vpool)] + index_args(hip, P), outs=(0, 1), **P.spec())
    P.rows, P.len, P.table = rows, ln, table
    assert np.array_equal(attn(hip, P, q, kpool, vpool, 0.125), good)
    check_attn(P, q, kpool, vpool, good, 0.125)


def test_paged_far_pages(hip):
    """Pages whose bytes lie past 4 GiB of their pool."""
    say("case: pages past 4 GiB")
    P = Paged([(1, 40)], DT_BF16, 16, 8, 8, 128, 256)
    far = (5 << 30) // (8 * 256 * 256) + 3
    x, q = P.make_x(), O.encode(P.rng.standard_normal((1, 8, 128)).astype(np.float32), DT_BF16)
    kpool, vpool = P.filled(), P.filled()
    blk = 8 * 256 * 256
    home = int(P.table[0, 0])
    bufs = []
    for pool in (kpool, vpool):
        b = hip.Buffer((far + 1) * blk)
        b.write(pool[home], far * blk)
        bufs.append(b)
    P.table[0, 0] = far
    want, _, _ = append(hip, Paged([(1, 40)], DT_BF16, 16, 8, 8, 128, 256), x, kpool, vpool)
    npages, P.npages = P.npages, far + 1
    qo, out = kept(hip, 8 * 128 * 2), kept(hip, 8 * 128 * 2)
    kw = P.spec(h=8, scale=0.09)
    ws = kept(hip, hip.attn_paged_ws(**kw))
    hip.builtin("attn_paged", [out, up(hip, q)] + bufs + index_args(hip, P) + [ws], **kw)
    P.table[0, 0], P.npages = home, npages
    check_attn(P, q, kpool, vpool, out.read(np.uint16).reshape(1, 8, 128), 0.09)
    P.table[0, 0], P.npages = far, far + 1
    hip.builtin("kv_append", [qo] + bufs + [up(hip, x)] + index_args(hip, P), outs=(0, 1, 2), **P.spec(h=8))
    assert np.array_equal(qo.read(np.uint16).reshape(1, 8, 128), want)
    kk, vv = kept(hip, 8 * 128 * 2), kept(hip, 8 * 128 * 2)
    hip.builtin("kv_read", [kk, vv] + bufs + index_args(hip, P), outs=(0, 1), **P.spec())
    assert np.array_equal(kk.read(np.uint16), x[0, 8 * 128:16 * 128])
    assert np.array_equal(vv.read(np.uint16), x[0, 16 * 128:])
    for b in bufs:
        b.free()


@pytest.mark.parametrize("bits", [16, 4])
def test_paged_requests_token_by_token(hip, bits):
    """Three requests of different lengths served together: prompts in one ragged
    call, then tokens in a captured graph whose lengths the host moves between the
    replays; every step equals the formulas over the rows appended so far, and the
    eager call bit for bit."""
    say(f"case: requests token by token, bits={bits}")
    H, K, hd, page, lens, steps = 8, 2, 128, 16, [37, 5, 90], 6
    full = Paged([(0, n + steps) for n in lens], DT_BF16, bits, H, K, hd, page)
    cos, sin = full.tables()
    rng = np.random.default_rng(9)
    gains = [(1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    kpool, vpool = full.stale(), full.stale()
    kb, vb, tb, lb = up(hip, kpool), up(hip, vpool), up(hip, full.table), up(hip, np.zeros(3, np.int32))
    cb, sb, gq, gk = up(hip, cos), up(hip, sin), up(hip, gains[0]), up(hip, gains[1])
    akw = dict(rope=2, norm=1, eps=float(np.float32(1e-5)))

    def shape(P):
        P.table, P.maxpages, P.npages = full.table, full.maxpages, full.npages
        return P

    def expect(P, x, q, out):
        for row, s, pos in P.each_row():
            qq, _, _, eq, _ = P.project(x, row, pos, np.float64, rope=2, norm=gains, eps=1e-5, cos=cos, sin=sin)
            assert near(O.decode(q[row], P.dt).astype(np.float64), qq, eq, P.dt)
            _, k, v, _, _ = P.project(x, row, pos, np.float32, rope=2, norm=gains, eps=1e-5, cos=cos, sin=sin)
            P.put(kpool, *P.where(s, pos), k)
            P.put(vpool, *P.where(s, pos), v)
        check_attn(P, q, kpool, vpool, out, 0.0884)

    P = shape(Paged([(n, n) for n in lens], DT_BF16, bits, H, K, hd, page))
    x = P.make_x()
    nb = P.n * H * hd * 2
    q, out, rows = kept(hip, nb), kept(hip, nb), up(hip, P.rows)
    lb.write(P.len)
    kw = P.spec(h=H, scale=0.0884)
    ws = hip.Buffer(hip.attn_paged_ws(**kw))
    hip.builtin("kv_append", [q, kb, vb, up(hip, x), tb, lb, rows, gq, gk, cb, sb], outs=(0, 1, 2), **P.spec(h=H, **akw))
    hip.builtin("attn_paged", [out, q, kb, vb, tb, lb, rows, ws], **kw)
    expect(P, x, q.read(np.uint16).reshape(P.n, H, hd), out.read(np.uint16).reshape(P.n, H, hd))

    one = shape(Paged([(1, n + 1) for n in lens], DT_BF16, bits, H, K, hd, page))
    xb, q, out, out2 = hip.Buffer(3 * 12 * hd * 2), *(kept(hip, 3 * H * hd * 2) for _ in range(3))
    kw = one.spec(h=H, scale=0.0884)
    ws = hip.Buffer(hip.attn_paged_ws(**kw))

    def step(o):
        hip.builtin("kv_append", [q, kb, vb, xb, tb, lb, gq, gk, cb, sb], outs=(0, 1, 2), **one.spec(h=H, **akw))
        hip.builtin("attn_paged", [o, q, kb, vb, tb, lb, ws], **kw)

    jit = hip.Jit()
    for i in range(steps):
        one.seqs = [(1, n + 1 + i) for n in lens]
        one.len = np.array([t for _, t in one.seqs], np.int32)
        x = one.make_x()
        xb.write(x)
        lb.write(one.len)
        if i == 0:
            with jit:
                step(out)
        jit.replay()
        got = out.read(np.uint16).reshape(3, H, hd)
        expect(one, x, q.read(np.uint16).reshape(3, H, hd), got)
        step(out2)
        assert np.array_equal(out2.read(np.uint16).reshape(3, H, hd), got), i
    assert np.array_equal(kb.read(np.uint8).reshape(kpool.shape), kpool)
    assert np.array_equal(vb.read(np.uint8).reshape(vpool.shape), vpool)
    jit.drop()


def test_attn_paged_equals_attn_over_a_contiguous_cache(hip):
    """The same rows in a contiguous cache through the attn builtin."""
    say("case: attn_paged against attn")
    P = Paged([(1, 200), (1, 200)], DT_BF16, 16, 8, 2, 128, 32)
    q = O.encode(P.rng.standard_normal((2, 8, 128)).astype(np.float32), DT_BF16)
    kpool, vpool = P.filled(), P.filled()
    got = O.decode(attn(hip, P, q, kpool, vpool, 0.09), DT_BF16).astype(np.float64)
    cache = []
    for pool in (kpool, vpool):
        c = np.zeros((2, 2, 256, 128))
        for s in range(2):
            for pos in range(200):
                c[s, :, pos] = P.get(pool, *P.where(s, pos))
        cache.append(up(hip, O.encode(c.astype(np.float32), DT_BF16)))
    out = hip.Buffer(2 * 8 * 128 * 2)
    hip.builtin("attn", [out, up(hip, q)] + cache + [up(hip, np.array([200], np.int32)), hip.Buffer(1 << 20)],
                b=2, h=8, hkv=2, hd=128, maxseq=256, qt=12, ct=12, ot=12, scale=0.09)
    want = O.decode(out.read(np.uint16), DT_BF16).reshape(2, 8, 128).astype(np.float64)
    for row, s, pos in P.each_row():
        _, tol = P.attend(q, P.held(kpool), P.held(vpool), row, s, pos, 0.09)
        assert near(got[row], want[row], tol + 2.0 ** -8 * np.abs(want[row]), DT_BF16)


@pytest.mark.parametrize("kernel,drop,word", [
    ("kv_append", dict(hd=80), "hd must"), ("kv_read", dict(page=48), "power of two"), ("attn_paged", dict(bits=8), "bits"),
    ("attn_paged", dict(dt=13), "dt must"), ("kv_append", dict(h=3), "multiple of hkv"), ("kv_append", dict(rope=3), "rope"),
    ("kv_append", dict(ldx=100), "ldx"), ("kv_append", dict(ldx=520 + 4), "ldx"), ("attn_paged", dict(n=5), "divide"),
    ("attn_paged", dict(npages=4000), "holds"), ("kv_read", dict(maxpages=300), "holds"), ("kv_read", dict(n=1 << 23), "rows"),
    ("attn_paged", dict(b=5000, n=5000), "sequences"), ("kv_append", dict(maxpages=1 << 27), "positions")])
def test_paged_refusals(hip, kernel, drop, word, monkeypatch):
    monkeypatch.setenv("THVM_HIP_QUIET", "1")
    P = Paged([(1, 9), (1, 4)], DT_BF16, 16, 4, 2, 64, 16)
    kpool = P.stale()
    a, k, v = hip.Buffer(2 * 8 * 64 * 2), up(hip, kpool), up(hip, kpool)
    idx = index_args(hip, P)
    kw = P.spec(h=4, scale=0.1)
    args = {"kv_append": [hip.Buffer(2 * 4 * 64 * 2), k, v, a] + idx, "kv_read": [hip.Buffer(512), hip.Buffer(512), k, v] + idx,
            "attn_paged": [hip.Buffer(2 * 4 * 64 * 2), a, k, v] + idx + [hip.Buffer(hip.attn_paged_ws(**kw))]}[kernel]
    outs = {"kv_append": (0, 1, 2), "kv_read": (0, 1), "attn_paged": (0,)}[kernel]
    hip.builtin(kernel, args, outs=outs, **kw)
    with pytest.raises(hip.ThvmHipError, match=word):
        hip.builtin(kernel, args, outs=outs, **{**kw, **drop})


def test_paged_refuses_shared_and_unaligned_buffers(hip, monkeypatch):
    monkeypatch.setenv("THVM_HIP_QUIET", "1")
    P = Paged([(1, 9), (1, 4)], DT_BF16, 16, 4, 2, 64, 16)
    k, v, x = up(hip, P.stale()), up(hip, P.stale()), hip.Buffer(2 * 8 * 64 * 2)
    q = hip.Buffer(2 * 4 * 64 * 2)
    idx, kw = index_args(hip, P), P.spec(h=4, scale=0.1)
    ws = hip.Buffer(hip.attn_paged_ws(**kw))
    for name, args, outs in (("kv_append", [x, k, v, x] + idx, (0, 1, 2)), ("kv_append", [q, k, k, x] + idx, (0, 1, 2)),
                             ("attn_paged", [q, q, k, v] + idx + [ws], (0,)), ("attn_paged", [q, x, k, v] + idx + [k], (0,))):
        with pytest.raises(hip.ThvmHipError, match="shares bytes|holds"):
            hip.builtin(name, args, outs=outs, **kw)
    view = hip.lib().thvm_hip_buf_view(x.id, 2, 2 * 8 * 64 * 2 - 2)
    with pytest.raises(hip.ThvmHipError, match="aligned"):
        hip.builtin("attn_paged", [q, view, k, v] + idx + [ws], **kw)
    with pytest.raises(hip.ThvmHipError, match="argument slot"):
        hip.builtin("attn_paged", [q, x, k, v] + idx, **kw)
