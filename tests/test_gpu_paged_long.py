"""The paged cache on the GPU where calls are long, wide or mixed: contexts that
many blocks share, batches of more sequences than a wave has lanes, pages of 256
and 1024 rows, prompts over long caches, row offsets that overlap, graphs that
share a workspace, and appends of many rows.  Tolerances are those of _paged_ref."""
import numpy as np
import pytest

import _oracle as O
from _paged_ref import DT_BF16, DT_F16, Paged, near
from test_gpu_paged import append, attn, check_append, check_attn, index_args, kept, say, up

pytestmark = pytest.mark.gpu


def random_pool(P):
    """A pool with a value in every slot."""
    if P.bits == 16:
        v = P.rng.standard_normal((P.npages, P.Hkv, P.page * P.hd)).astype(np.float32)
        return O.encode(v, P.dt).view(np.uint8).reshape(P.npages, P.Hkv, P.page * P.rb)
    pool = P.rng.integers(0, 256, (P.npages, P.Hkv, P.page * P.rb)).astype(np.uint8)
    scales = pool[..., P.page * P.hd // 2:]
    scales[...] = 122 + scales % 5                  # 2^-5 to 2^-1
    return pool


def case(seqs, dt, bits, H, Hkv, hd, page, pages=None, **kw):
    """A Paged; `pages`: its sequences share so many physical pages, at random."""
    P = Paged(seqs, dt, bits, H, Hkv, hd, page, **kw)
    if pages:
        P.npages = pages
        P.table = np.where(P.table >= 0, P.rng.integers(0, pages, P.table.shape), -1).astype(np.int32)
    q = O.encode((1.5 * P.rng.standard_normal((P.n, H, hd))).astype(np.float32), dt)
    return P, q, random_pool(P), random_pool(P), np.float32(hd ** -0.5)


LONG = {"one": [(1, 20000)], "two": [(1, 9000), (1, 70)], "rows": [(2, 5000), (1, 300), (3, 3)],
        "four": [(4, 2100), (4, 4000)]}


@pytest.mark.parametrize("dt,bits", [(DT_BF16, 16), (DT_F16, 4)])
@pytest.mark.parametrize("H,Hkv,hd,page", [(8, 1, 128, 16), (16, 1, 64, 64), (32, 2, 128, 256), (3, 3, 64, 1024),
                                           (40, 10, 64, 128)])
@pytest.mark.parametrize("seqs", LONG)
def test_attn_paged_long_contexts(hip, dt, bits, H, Hkv, hd, page, seqs):
    say(f"case: attn_paged long contexts dt={dt} bits={bits} H={H} Hkv={Hkv} hd={hd} page={page} {seqs}")
    P, q, kp, vp, scale = case(LONG[seqs], dt, bits, H, Hkv, hd, page)
    check_attn(P, q, kp, vp, attn(hip, P, q, kp, vp, scale, t=max(r for r, _ in P.seqs)), scale)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("H,Hkv,hd", [(4, 1, 128), (2, 2, 64), (16, 1, 64)])
@pytest.mark.parametrize("seqs", [[(1, 37 * i % 900 + 1) for i in range(130)], [(1, 600)] * 65,
                                  [(i % 3, 53 * i % 700 + 3) for i in range(100)]], ids=["b130", "even65", "ragged100"])
def test_attn_paged_wide_batches(hip, bits, H, Hkv, hd, seqs):
    """More sequences than a wave has lanes, each of several chunks or one."""
    say(f"case: attn_paged wide bits={bits} H={H} Hkv={Hkv} hd={hd} b={len(seqs)}")
    P, q, kp, vp, scale = case(seqs, DT_BF16, bits, H, Hkv, hd, 32)
    check_attn(P, q, kp, vp, attn(hip, P, q, kp, vp, scale), scale)


@pytest.mark.parametrize("dt,bits,H,Hkv,hd,page", [(DT_BF16, 16, 4, 1, 64, 16), (DT_F16, 4, 4, 2, 128, 32)])
@pytest.mark.parametrize("b", [66, 257, 700, 4096])
def test_paged_many_requests(hip, dt, bits, H, Hkv, hd, page, b):
    """Hundreds of requests in one ragged call, tokens beside prompts and empty ones:
    appended, read back and attended."""
    say(f"case: paged b={b} dt={dt} bits={bits} H={H} Hkv={Hkv} hd={hd}")
    n = [0 if i % 7 == 3 else 40 if i % 97 == 65 else 1 + (i % 5 == 0) for i in range(b)]
    P, q, kp, vp, scale = case([(r, r + 29 * i % 300 + 700 * (i % 59 == 1)) for i, r in enumerate(n)], dt, bits, H, Hkv,
                               hd, page, extra=2)
    x = P.make_x()
    got = append(hip, P, x, kp, vp)
    check_append(P, x, kp, vp, got)
    check_attn(P, q, got[1], got[2], attn(hip, P, q, got[1], got[2], scale), scale)
    check_attn(P, q, got[1], got[2], attn(hip, P, q, got[1], got[2], scale, t=40), scale)
    k, v = (kept(hip, P.n * Hkv * hd * 2) for _ in range(2))
    hip.builtin("kv_read", [k, v, up(hip, got[1]), up(hip, got[2])] + index_args(hip, P), outs=(0, 1), **P.spec())
    kheld = P.held(got[1])
    k = O.decode(k.read(np.uint16).reshape(P.n, Hkv, hd), dt).astype(np.float64)
    for row, s, pos in P.each_row():
        pg, slot = P.where(s, pos)
        assert np.array_equal(k[row], kheld[pg, :, slot]), (row, s, pos)


def test_attn_paged_garbage_of_many_requests(hip):
    """Offsets, lengths and pages of hundreds of requests full of garbage: the calls
    end inside their buffers, and a good one after them is right."""
    say("case: garbage of many requests")
    rng = np.random.default_rng(8)
    P, q, kp, vp, scale = case([(1 + i % 3, 20 + 7 * i % 400) for i in range(300)], DT_BF16, 16, 4, 1, 64, 16)
    good = attn(hip, P, q, kp, vp, scale)
    rows, ln, table = P.rows.copy(), P.len.copy(), P.table.copy()
    for i in range(5):
        P.rows = rng.integers(-2 ** 31, 2 ** 31, rows.shape).astype(np.int32) if i % 2 else rng.permutation(rows)
        P.len = rng.integers(-2 ** 31, 2 ** 31, ln.shape).astype(np.int32) if i % 3 else ln
        P.table = rng.integers(-2 ** 31, 2 ** 31, table.shape).astype(np.int32) if i % 4 > 1 else table
        attn(hip, P, q, kp, vp, scale)
        append(hip, P, P.make_x(), kp, vp)
    P.rows, P.len, P.table = rows, ln, table
    assert np.array_equal(attn(hip, P, q, kp, vp, scale), good)
    check_attn(P, q, kp, vp, good, scale)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("b,ctx", [(24, 16000), (9, 70000)])
def test_attn_paged_twice_the_chunks(hip, bits, b, ctx):
    """Much cache, of lengths that the first plan divides badly.  The sequences share
    pages; a few of them are checked."""
    say(f"case: attn_paged b={b} ctx={ctx} bits={bits}")
    P, q, kp, vp, scale = case([(1, ctx - 100 * i) for i in range(b)], DT_F16, bits, 8, 8, 64, 64, pages=60)
    g = O.decode(attn(hip, P, q, kp, vp, scale), DT_F16).astype(np.float64)
    kheld, vheld = P.held(kp), P.held(vp)
    assert np.isfinite(g).all()
    for row, s, pos in P.each_row():
        if s % 4 == 1:
            want, tol = P.attend(q, kheld, vheld, row, s, pos, scale)
            assert near(g[row], want, tol, DT_F16), row


@pytest.mark.parametrize("dt,bits,hd,page", [(DT_BF16, 16, 128, 32), (DT_F16, 4, 64, 64)])
@pytest.mark.parametrize("H,Hkv,rows", [(32, 2, 1), (4, 2, 7), (80, 2, 1)])
def test_attn_paged_merged_columns(hip, dt, bits, hd, page, H, Hkv, rows):
    """Tiles of 16 columns, many of them, in a few chunks each."""
    say(f"case: attn_paged merged columns dt={dt} bits={bits} hd={hd} H={H} rows={rows}")
    P, q, kp, vp, scale = case([(rows, max(rows, 4000 - 97 * i)) for i in range(40)], dt, bits, H, Hkv, hd, page, pages=70)
    check_attn(P, q, kp, vp, attn(hip, P, q, kp, vp, scale), scale)


def test_attn_paged_heads_each_their_own(hip):
    """Hundreds of kv heads."""
    say("case: attn_paged of 512 kv heads")
    P, q, kp, vp, scale = case([(1, 700), (1, 33), (1, 1)], DT_BF16, 16, 512, 512, 64, 64)
    check_attn(P, q, kp, vp, attn(hip, P, q, kp, vp, scale), scale)


PROMPT = {"chunk": [(150, 2500)], "chunks": [(70, 1900), (129, 129), (1, 800), (33, 40)], "even": [(40, 640), (40, 900)]}


@pytest.mark.parametrize("dt,bits", [(DT_BF16, 16), (DT_BF16, 4), (DT_F16, 16), (DT_F16, 4)])
@pytest.mark.parametrize("H,Hkv,hd,page", [(4, 1, 64, 16), (5, 5, 128, 256), (2, 2, 64, 1024), (6, 2, 128, 16)])
@pytest.mark.parametrize("seqs", PROMPT)
def test_attn_paged_prompts_over_long_caches(hip, dt, bits, H, Hkv, hd, page, seqs):
    say(f"case: attn_paged prompts dt={dt} bits={bits} H={H} Hkv={Hkv} hd={hd} page={page} {seqs}")
    P, q, kp, vp, scale = case(PROMPT[seqs], dt, bits, H, Hkv, hd, page)
    check_attn(P, q, kp, vp, attn(hip, P, q, kp, vp, scale), scale)


def test_attn_paged_offsets_that_overlap(hip):
    """More tiles than rows can have: the call ends, stays in its buffers, and the
    good calls after it are right."""
    say("case: attn_paged offsets that overlap")
    few = case([(1, 900), (0, 5), (2, 700), (0, 9), (1, 300), (0, 1), (0, 1), (0, 1)], DT_BF16, 16, 4, 1, 64, 16)
    many = case([(40, 900), (30, 300), (0, 7), (0, 600)], DT_BF16, 16, 4, 1, 64, 16)
    good = [attn(hip, *c) for c in (few, many)]
    for P, q, kp, vp, scale in (few, many):
        rows = P.rows
        for i in range(4):
            P.rows = np.where(np.arange(P.b + 1) % 2 == i % 2, 0, P.n if i < 2 else 3).astype(np.int32)
            attn(hip, P, q, kp, vp, scale)
        P.rows = rows
    for (P, q, kp, vp, scale), first in zip((few, many), good):
        again = attn(hip, P, q, kp, vp, scale)
        assert np.array_equal(again, first)
        check_attn(P, q, kp, vp, again, scale)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("page", [16, 128])
def test_paged_far_pages_of_prompts(hip, bits, page):
    """A prompt's rows in pages past 4 GiB of their pool: appended, read and attended."""
    say(f"case: a prompt's pages past 4 GiB, bits={bits} page={page}")
    P, q, kp, vp, scale = case([(40, 90), (17, 17)], DT_BF16, bits, 8, 8, 128, page)
    x = P.make_x()
    want = append(hip, P, x, kp, vp)
    ref = attn(hip, P, q, want[1], want[2], scale)
    check_attn(P, q, want[1], want[2], ref, scale)
    blk = 8 * page * P.rb
    far, near_, n0 = (5 << 30) // blk, P.table.copy(), P.npages
    bufs = []
    for pool in (kp, vp):
        bufs.append(hip.Buffer((far + n0) * blk))
        bufs[-1].write(pool, far * blk)
    P.table, P.npages = np.where(near_ >= 0, near_ + far, near_).astype(np.int32), far + n0
    ix = index_args(hip, P)
    qo, out, k, v = (kept(hip, P.n * 8 * 128 * 2) for _ in range(4))
    kw = P.spec(h=8, scale=float(scale))
    hip.builtin("kv_append", [qo] + bufs + [up(hip, x)] + ix, outs=(0, 1, 2), **P.spec(h=8))
    hip.builtin("attn_paged", [out, up(hip, q)] + bufs + ix + [kept(hip, hip.attn_paged_ws(**kw))], **kw)
    hip.builtin("kv_read", [k, v] + bufs + ix, outs=(0, 1), **P.spec())
    assert np.array_equal(qo.read(np.uint16).reshape(want[0].shape), want[0])
    assert np.array_equal(out.read(np.uint16).reshape(ref.shape), ref)
    P.table, P.npages = near_, n0
    for got, pool in ((k, want[1]), (v, want[2])):
        held, got = P.held(pool), O.decode(got.read(np.uint16).reshape(P.n, 8, 128), DT_BF16).astype(np.float64)
        for row, s, pos in P.each_row():
            pg, slot = P.where(s, pos)
            assert np.array_equal(got[row], held[pg, :, slot]), row
    for b in bufs:
        b.free()


def test_attn_paged_graphs_share_a_workspace(hip):
    """Two captured calls, one of single tokens and one of prompts, in one workspace,
    replayed in turn with eager calls and lengths that move between them."""
    say("case: graphs that share a workspace")
    one = case([(1, 4000), (1, 700), (1, 64)], DT_BF16, 16, 8, 2, 128, 64)
    two = case([(80, 3000), (1, 2000), (20, 20)], DT_BF16, 4, 8, 2, 128, 32)
    wide = case([(16, 3000)], DT_BF16, 16, 8, 8, 64, 64)
    runs, need = [], max(hip.attn_paged_ws(**c[0].spec(h=8, scale=float(c[4]))) for c in (one, two, wide))
    ws = kept(hip, need)
    for P, q, kp, vp, scale in (one, two, wide):
        out = kept(hip, P.n * 8 * P.hd * 2)
        ix = index_args(hip, P)
        runs.append((P, out, ix[1], [out, up(hip, q), up(hip, kp), up(hip, vp)] + ix + [ws], P.spec(h=8, scale=float(scale))))
    jits = []
    for _, _, _, args, kw in runs[:2]:
        jit = hip.Jit()
        with jit:
            hip.builtin("attn_paged", args, **kw)
        jits.append(jit)
    for i in range(4):
        for (P, q, kp, vp, scale), (_, out, lb, args, kw), jit in zip((one, two), runs, jits):
            full = P.seqs
            P.seqs = [(r, t - i * (t > 100)) for r, t in full]
            P.len = np.array([t for _, t in P.seqs], np.int32)
            lb.write(P.len)
            jit.replay()
            got = out.read(np.uint16).reshape(P.n, 8, P.hd)
            check_attn(P, q, kp, vp, got, scale)
            hip.builtin("attn_paged", runs[2][3], **runs[2][4])
            hip.builtin("attn_paged", args, **kw)
            assert np.array_equal(out.read(np.uint16).reshape(P.n, 8, P.hd), got), i
            P.seqs = full
    check_attn(wide[0], wide[1], wide[2], wide[3], runs[2][1].read(np.uint16).reshape(16, 8, 64), wide[4])
    for jit in jits:
        jit.drop()


@pytest.mark.parametrize("dt", [DT_BF16, DT_F16])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("H,Hkv,hd,page,rope,norm", [(16, 4, 128, 32, 2, True), (6, 3, 128, 16, 1, False),
                                                     (12, 12, 64, 256, 1, True), (3, 3, 64, 64, 2, False)])
def test_kv_append_many_rows(hip, dt, bits, H, Hkv, hd, page, rope, norm):
    groups = -(-(H + 2 * Hkv) // (512 // hd))
    n = 8192 // groups + 5
    say(f"case: kv_append rows={n} dt={dt} bits={bits} H={H} Hkv={Hkv} hd={hd} page={page}")
    P = Paged([(n // 2, n // 2 + 9), (1, 70), (n - n // 2 - 1, n)], dt, bits, H, Hkv, hd, page, extra=2)
    x, kp, vp = P.make_x(), P.stale(), P.stale()
    kw = dict(rope=rope, **dict(zip(("cos", "sin"), P.tables())))
    if norm:
        kw.update(norm=[(1 + 0.1 * P.rng.standard_normal(hd)).astype(np.float32) for _ in range(2)], eps=1e-5)
    check_append(P, x, kp, vp, append(hip, P, x, kp, vp, **kw), **kw)


@pytest.mark.parametrize("dt,bits,Hkv,hd,page", [(DT_BF16, 16, 8, 128, 64), (DT_F16, 4, 6, 128, 32),
                                                 (DT_BF16, 4, 20, 64, 16), (DT_F16, 16, 9, 64, 256)])
def test_kv_read_many_rows(hip, dt, bits, Hkv, hd, page):
    n = 8192 // -(-2 * Hkv // (512 // hd)) + 3
    say(f"case: kv_read rows={n} dt={dt} bits={bits} Hkv={Hkv} hd={hd} page={page}")
    P = Paged([(n - 40, n), (40, 77)], dt, bits, Hkv, Hkv, hd, page, holes=((0, 3, -1),))
    kp, vp = random_pool(P), random_pool(P)
    k, v = (kept(hip, n * Hkv * hd * 2) for _ in range(2))
    hip.builtin("kv_read", [k, v, up(hip, kp), up(hip, vp)] + index_args(hip, P), outs=(0, 1), **P.spec())
    kheld, vheld = P.held(kp), P.held(vp)
    k, v = (O.decode(z.read(np.uint16).reshape(n, Hkv, hd), dt).astype(np.float64) for z in (k, v))
    for row, s, pos in P.each_row():
        at = P.where(s, pos)
        for got, held in ((k, kheld), (v, vheld)):
            assert np.array_equal(got[row], held[at[0], :, at[1]] if at else np.zeros((Hkv, hd))), (row, s, pos)
