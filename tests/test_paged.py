"""CPU side of the paged cache: the 4-bit format's reference against its
definition, the specs that the builtins refuse, and the index functions of the
kernels, compiled for the host, over garbage rows, lengths and page tables."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

from _paged_ref import DT_BF16, DT_F16, E2M1, Paged, quantise, values

ROOT = Path(__file__).resolve().parents[1]
SPEC = dict(n=4, b=2, h=8, hkv=2, hd=64, page=16, maxpages=5, npages=9, scale=0.125)


@pytest.mark.parametrize("dt,lo,hi", [(DT_BF16, -126, 125), (DT_F16, -23, 13)])
def test_four_bit_reference(dt, lo, hi):
    """Each value goes to a nearest one of the 15, the scale is the smallest that
    holds the largest, and held values come back unchanged."""
    rng = np.random.default_rng(1)
    y = (rng.standard_normal((200, 64)) * 2.0 ** rng.integers(-40, 15, (200, 1))).astype(np.float32)
    y[0], y[1, :32], y[2, 5] = 0, 6 * 2.0 ** 3, 6.0000005 * 2.0 ** 20
    c, s = quantise(y, dt)
    v = values(c, s)
    e = s.astype(int) - 127
    amax = np.abs(y).reshape(200, 2, 32).max(-1).astype(np.float64)
    assert ((e >= lo) & (e <= hi)).all()
    free = (e > lo) & (e < hi)
    assert (amax[free] <= 6 * 2.0 ** e[free]).all() and (amax[free] > 6 * 2.0 ** (e[free] - 1)).all()
    unit = np.repeat(2.0 ** e, 32, -1)
    best = np.abs(y.astype(np.float64)[..., None] - E2M1 * unit[..., None]).min(-1)
    assert np.array_equal(np.abs(y - v), best)
    c2, s2 = quantise(v.astype(np.float32), dt)
    assert np.array_equal(values(c2, s2), v)
    x = np.zeros((3, 32), np.float32)
    x[0, 3], x[1, 0], x[2, 31] = np.nan, np.inf, -np.inf
    c, s = quantise(x, dt)
    assert (s == 255).all() and np.isnan(values(c, s)).all()


def test_ties_go_to_the_even_code():
    b = np.array([6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5.0] * 4, np.float32)
    assert quantise(b, DT_BF16)[0][:8].tolist() == [7, 0, 2, 2, 4, 4, 6, 6]


@pytest.fixture(scope="module")
def lib():
    import thvm_amd
    if not thvm_amd.LIB_PATH.exists():
        from thvm_amd import build
        build.build(verbose=False)
    return thvm_amd


def test_workspace_needs_no_device(lib):
    assert lib.attn_paged_ws(**SPEC) >= 16
    assert lib.attn_paged_ws(**{**SPEC, "n": 4096, "b": 64, "ragged": 1}) >= 16


@pytest.mark.parametrize("bad,word", [
    (dict(hd=96), "hd must"), (dict(hd=0), "hd must"), (dict(dt=13), "dt must"), (dict(bits=8), "bits"),
    (dict(page=24), "power of two"), (dict(page=8), "power of two"), (dict(page=2048), "power of two"),
    (dict(b=0), "sequences"), (dict(b=4097, n=4097), "sequences"), (dict(n=0), "rows"), (dict(n=(1 << 22) + 2), "rows"),
    (dict(n=5), "divide"), (dict(ragged=2), "ragged"), (dict(maxpages=0), "positions"),
    (dict(maxpages=(1 << 26) + 1), "positions"), (dict(npages=0), "positions"), (dict(npages=1 << 31), "positions"),
    (dict(hkv=0), "hkv"), (dict(hkv=2000, h=2000), "hkv"), (dict(h=0), "multiple"), (dict(h=7), "multiple"),
    (dict(h=2048, hkv=2), "multiple"), (dict(n=1 << 22, h=64), "heads"), (dict(n=4096, b=4096, hkv=256, h=256), "2.19"), (dict(t=0), "t=0"), (dict(t=1), "t=1"),
    (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale")])
def test_attn_paged_specs_refused(lib, bad, word, monkeypatch):
    monkeypatch.setenv("THVM_HIP_QUIET", "1")
    with pytest.raises(lib.ThvmHipError, match=word):
        lib.attn_paged_ws(**{**SPEC, **bad})


def test_attn_paged_ws_wants_its_own_program(lib, monkeypatch):
    monkeypatch.setenv("THVM_HIP_QUIET", "1")
    for program in (None, b"", b"attn_paged n=1", b"thvm-builtin:kv_read n=1", b"thvm-builtin:attn_paged n=1",
                    b"thvm-builtin:attn_paged n"):
        assert lib.lib().thvm_hip_attn_paged_ws(program) == 0
        assert lib.last_error()


class Args(C.Structure):
    """ThvmPagedArgs (kern_api.h)."""
    _fields_ = [(n, C.c_void_p) for n in ("q", "out", "kpages", "vpages", "x", "k", "v", "table", "len", "rows", "gq",
                                          "gk", "cos_t", "sin_t", "ws")] + \
        [(n, C.c_uint32) for n in ("n", "b", "H", "Hkv", "hd", "page", "maxpages", "npages", "dt", "bits", "ragged",
                                   "rope", "norm", "ldx", "t")] + [("eps", C.c_float), ("scale", C.c_float)]


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    """The checks and the index functions, compiled for the host."""
    d = tmp_path_factory.mktemp("paged")
    (d / "h.c").write_text('''
#include "paged_index.h"
int chk(const ThvmPagedArgs *a, int op, char *err) { return pg_check(a, op, err, 200); }
void seq(const ThvmPagedArgs *a, uint32_t s, int32_t *o) { PgSeq q = pg_seq(a, s); o[0] = q.r0; o[1] = q.r1; o[2] = q.len; }
int32_t page(const ThvmPagedArgs *a, uint32_t s, int32_t p) { return pg_page(a, s, p); }
uint64_t block(const ThvmPagedArgs *a, int32_t id, uint32_t h) { return pg_block(a, id, h); }
uint32_t bbytes(const ThvmPagedArgs *a) { return pg_block_bytes(a); }
uint64_t pool(const ThvmPagedArgs *a) { return pg_pool_bytes(a); }
uint64_t size(void) { return sizeof(ThvmPagedArgs); }
''')
    subprocess.run(["gcc", "-std=c11", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__",
                    "-I/opt/rocm/include", f"-I{ROOT / 'include'}", f"-I{ROOT / 'thvm_amd' / 'csrc'}", str(d / "h.c"),
                    "-o", str(d / "h.so")], check=True)
    L = C.CDLL(str(d / "h.so"))
    for f in ("block", "pool", "size"):
        getattr(L, f).restype = C.c_uint64
    assert L.size() == C.sizeof(Args)
    return L


def args(**kw):
    a = Args(**{**dict(n=6, b=2, H=4, Hkv=2, hd=64, page=16, maxpages=5, npages=9, dt=12, bits=16, ldx=512, t=3,
                       eps=1e-6, scale=0.1), **kw})
    return a


@pytest.mark.parametrize("op,bad,word", [
    (0, dict(rope=3), "rope"), (0, dict(norm=2), "norm"), (0, dict(norm=1, eps=-1.0), "eps"),
    (0, dict(norm=1, eps=float("nan")), "eps"), (0, dict(ldx=511), "ldx"), (0, dict(ldx=516), "ldx"), (0, dict(H=5), "multiple"),
    (0, dict(hd=32), "hd must"), (1, dict(page=17), "power of two"), (1, dict(bits=2), "bits"), (1, dict(n=7), "divide"),
    (1, dict(n=1 << 22, Hkv=8), "heads"), (2, dict(t=2), "t=2"), (2, dict(dt=9), "dt must")])
def test_shapes_refused(host, op, bad, word):
    err = C.create_string_buffer(200)
    assert host.chk(C.byref(args()), op, err) == 0
    assert host.chk(C.byref(args(**bad)), op, err) == -1
    assert word in err.value.decode()


@pytest.mark.parametrize("bits", [16, 4])
def test_indexes_of_garbage_stay_inside(host, bits):
    """Whatever rows, len and table hold: rows lie in [0, n] in order, lengths in
    [0, 2^30], a page's blocks inside the pool."""
    rng = np.random.default_rng(2)
    o = (C.c_int32 * 3)()
    edge = np.array([-2 ** 31, -1, 0, 1, 5, 6, 7, 2 ** 31 - 1, 2 ** 30, 8, 9, 80], np.int64)
    for _ in range(300):
        pick = lambda k: np.where(rng.random(k) < 0.5, rng.choice(edge, k), rng.integers(-2 ** 31, 2 ** 31, k)).astype(np.int32)  # noqa: E731
        rows, ln, table = pick(3), pick(2), pick(10)
        a = args(bits=bits, ragged=1, rows=rows.ctypes.data, len=ln.ctypes.data, table=table.ctypes.data)
        for s in range(2):
            host.seq(C.byref(a), s, o)
            r0, r1, length = o
            assert 0 <= r0 <= r1 <= 6 and 0 <= length <= 2 ** 30
            for i in range(r0, r1):
                assert -2 ** 31 <= length - (r1 - i) < 2 ** 31
            for pos in (-2 ** 31, -1, 0, 15, 16, 79, 80, 2 ** 30, 2 ** 31 - 1, int(rng.integers(0, 80))):
                p = host.page(C.byref(a), s, C.c_int32(pos))
                assert -1 <= p < 9
                if p >= 0:
                    assert 0 <= pos < 80 and table[s * 5 + pos // 16] == p
                    for h in range(2):
                        assert host.block(C.byref(a), p, h) + host.bbytes(C.byref(a)) <= host.pool(C.byref(a))
    a = args(bits=bits, len=ln.ctypes.data)
    host.seq(C.byref(a), 1, o)
    assert (o[0], o[1]) == (3, 6)


def test_blocks_past_four_gib(host):
    a = args(npages=1 << 20, Hkv=8, hd=128, page=256)
    assert host.block(C.byref(a), (1 << 20) - 1, 7) == ((1 << 20) * 8 - 1) * 256 * 256


def test_reference_holds_what_it_puts():
    for bits in (16, 4):
        P = Paged([(3, 40), (1, 5)], DT_BF16, bits)
        pool = P.filled()
        held = P.held(pool)
        for s, t in ((0, 40), (1, 5)):
            for pos in range(t):
                page, slot = P.where(s, pos)
                assert np.array_equal(held[page, :, slot], P.get(pool, page, slot)) and np.isfinite(held[page, :, slot]).all()
        assert np.isnan(held).any()
