"""The paged-cache operators on real work: ``kv_append`` (q/k norms, position
rotation and the append), ``kv_read`` (a cache's rows as values) and
``attn_paged`` (attention of a ragged batch over the pages), caches of 16 or of
4 bits.

A case is a dict of plain values.  ``op`` is "append" (q and the pages; over 4
bits q and the appended rows as ``kv_read`` gives them) or "attn".  ``batch``
sequences have at most ``rows`` new rows over at most ``ctx`` rows that are in
the cache already; ``mix`` says how they differ: "even" (all at those numbers),
"ragged" (rows and contexts spread down from them), "mixed" (one sequence in
four at ``rows``, the others a single row each).  ``own`` is False for the plain
form in torch operations and True for the calls into the framework."""
from __future__ import annotations

import math
import random

import torch

own = False

_TORCH = {"bf16": torch.bfloat16, "fp16": torch.float16}
_DT = {"bf16": 12, "fp16": 11}


# ---- the cases --------------------------------------------------------------

def _case(name, **kw):
    c = dict(name=name, op="attn", heads=32, kv_heads=8, hd=128, dt="bf16", bits=16, page=64, batch=1, rows=1,
             ctx=2048, mix="even", rope=0, norm=False)
    c.update(kw)
    return c


def listed():
    return [
        # one user's token of a Llama-8B-shape layer: q rotated, k and v into the pages (launch latency)
        _case("append_b1", op="append", rope=1),
        # a serving batch's tokens at ragged positions, q and k normed per head, rotated in halves
        _case("append_b48_qknorm", op="append", heads=16, kv_heads=8, hd=64, dt="fp16", page=16, batch=48, ctx=3000,
              mix="ragged", rope=2, norm=True),
        # ragged prompts read in together
        _case("append_prompts", op="append", batch=6, rows=3000, ctx=500, mix="ragged", rope=1),
        # the same into a cache of 4 bits, and a batch of tokens into one
        _case("append_prompts_4bit", op="append", batch=4, rows=2048, ctx=0, mix="ragged", rope=2, norm=True, bits=4,
              page=128),
        _case("append_b64_4bit", op="append", batch=64, ctx=4000, mix="ragged", rope=1, bits=4, page=32),
        # one user's token over 2049 rows
        _case("attn_b1"),
        # GPT-2 XL's heads for eight users, at chat-sized contexts
        _case("attn_gpt2_xl_b8", heads=25, kv_heads=25, hd=64, dt="fp16", page=16, batch=8, ctx=1000, mix="ragged"),
        # a serving batch whose contexts run from hundreds of rows to many thousands
        _case("attn_b32_ragged", batch=32, ctx=16000, mix="ragged"),
        # two long documents held in 4 bits
        _case("attn_long_4bit", batch=2, ctx=100000, bits=4, page=128),
        # a speculative verify: four rows a sequence over 4 bits
        _case("attn_verify_b16_4bit", batch=16, rows=4, ctx=8000, mix="ragged", bits=4),
        # ragged prompts read in from nothing
        _case("attn_prompts", batch=5, rows=3001, ctx=0, mix="ragged"),
        # chunks of long prompts beside other users' single tokens, over 4 bits
        _case("attn_mixed_4bit", dt="fp16", batch=12, rows=512, ctx=12000, mix="mixed", bits=4, page=32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: any head layout, type, page size and mix, from single
    tokens to the listed prompts and contexts."""
    largest = {op: [max(work(c)[k] for c in listed() if c["op"] == op) for k in ("bytes", "flops")] for op in ("append", "attn")}
    while True:
        kv = rng.choice((1, 2, 4, 8, 8, 16))
        c = _case("", op=rng.choice(("append", "attn", "attn")), kv_heads=kv,
                  heads=kv * rng.choice([g for g in (1, 2, 3, 4, 5, 8, 16) if 4 <= g * kv <= 64]),
                  hd=rng.choice((64, 128, 128)), dt=rng.choice(("bf16", "bf16", "fp16")), bits=rng.choice((16, 4)),
                  page=rng.choice((16, 32, 64, 128, 256)), batch=_log(rng, 1, 64), mix=rng.choice(("even", "ragged", "mixed")))
        c["rows"] = 1 if rng.random() < 0.5 else _log(rng, 2, 3000)
        c["ctx"] = _log(rng, 1, 100000) - 1
        if c["op"] == "append":
            c.update(rope=rng.randint(0, 2), norm=rng.random() < 0.5)
        w = work(c)
        pad = c["batch"] * c["rows"] * c["heads"] * (c["rows"] + c["ctx"])       # the plain form's padded scores
        pool = c["batch"] * (c["rows"] + c["ctx"]) * c["kv_heads"] * c["hd"]
        if w["bytes"] <= largest[c["op"]][0] and w["flops"] <= largest[c["op"]][1] and pool <= 6e8 and \
                (c["op"] == "append" or pad <= 2e9):
            del c["name"]
            return c


def _lengths(c):
    """(new rows, cache rows with them) of each sequence, by the case alone."""
    rng = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    out = []
    for i in range(c["batch"]):
        n, ctx = c["rows"], c["ctx"]
        if c["mix"] != "even" and i:
            ctx = _log(rng, max(1, ctx // 64), max(1, ctx)) if ctx else 0
        if c["mix"] == "ragged" and i:
            n = rng.randint((n + 3) // 4, n)
        if c["mix"] == "mixed" and i % 4:
            n = 1
        out.append((n, n + ctx))
    return out


def _row_bytes(c):
    """Bytes of a cache row of one head: its 16-bit values, or codes and scales."""
    return c["hd"] * 2 if c["bits"] == 16 else c["hd"] // 2 + c["hd"] // 32


def work(case):
    c = case
    L = _lengths(c)
    n, io, kv = sum(r for r, _ in L), c["heads"] * c["hd"] * 2, c["kv_heads"] * c["hd"] * 2
    if c["op"] == "append":
        b = n * (io + 2 * kv) + n * io + n * 2 * c["kv_heads"] * _row_bytes(c)
        if c["bits"] == 4:                       # and read back as values
            b += n * 2 * c["kv_heads"] * _row_bytes(c) + n * 2 * kv
        return {"bytes": b, "flops": 8.0 * n * (c["heads"] + c["kv_heads"]) * c["hd"]}
    seen = sum(r * (t - r) + r * (r + 1) / 2 for r, t in L)
    return {"bytes": 2 * n * io + sum(t for _, t in L) * 2 * c["kv_heads"] * _row_bytes(c),
            "flops": 4.0 * seen * c["heads"] * c["hd"]}


# ---- the inputs of a case, from the seed alone -------------------------------

def _plan(c):
    """Whole numbers of a case: lengths, page tables, and the sizes they give."""
    L = _lengths(c)
    need = [-(-t // c["page"]) for _, t in L]
    return {"L": L, "need": need, "n": sum(r for r, _ in L), "maxpages": max(need) + 1, "npages": sum(need) + 3,
            "most": max(t for _, t in L), "t": max(r for r, _ in L)}


def _inputs(c, seed):
    p = _plan(c)
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 11)

    def rnd(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    T, dt, H, K, hd = {}, _TORCH[c["dt"]], c["heads"], c["kv_heads"], c["hd"]
    pages = torch.randperm(p["npages"], generator=g, device="cuda").to(torch.int32)
    first = [sum(p["need"][:i]) for i in range(c["batch"])]
    at = torch.arange(p["maxpages"], device="cuda")
    have = torch.tensor(p["need"], device="cuda")[:, None]
    idx = torch.tensor(first, device="cuda")[:, None] + at
    T["table"] = torch.where(at < have, pages[idx.clamp(max=p["npages"] - 1)], -1).to(torch.int32)
    T["len"] = torch.tensor([t for _, t in p["L"]], device="cuda", dtype=torch.int32)
    T["rows"] = torch.tensor([0] + [r for r, _ in p["L"]], device="cuda").cumsum(0).to(torch.int32)
    block = (p["npages"], K, c["page"] * _row_bytes(c))
    for name in ("kpages", "vpages"):
        if c["op"] == "append":                   # a pool that held other requests before
            T[name] = torch.full(block, 0x11, device="cuda", dtype=torch.uint8)
        elif c["bits"] == 16:
            T[name] = rnd(p["npages"], K, c["page"] * hd).to(dt).view(torch.uint8).view(block)
        else:
            codes, scales = _quantise(rnd(p["npages"], K, c["page"], hd), c["dt"])
            T[name] = torch.cat((codes.flatten(2), scales.flatten(2)), 2)
    if c["op"] == "append":
        T["x"] = rnd(p["n"], (H + 2 * K) * hd).to(dt)
        if c["norm"]:
            T["gq"], T["gk"] = 1.0 + 0.1 * rnd(hd), 1.0 + 0.1 * rnd(hd)
        if c["rope"]:
            f = 500000.0 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
            a = torch.arange(p["maxpages"] * c["page"], device="cuda", dtype=torch.float64)[:, None] * f
            T["cos"], T["sin"] = a.cos().float(), a.sin().float()
    else:
        T["q"] = (1.5 * rnd(p["n"], H, hd)).to(dt)
    return p, T


# ---- the plain form ------------------------------------------------------------

def _step(amax, dt):
    """The scale of 32 values by their largest: its exponent e, 2^e the smallest
    power of two with amax <= 6 * 2^e, inside the range whose values all are
    numbers of the 16-bit type."""
    lo, hi = (-126, 125) if dt == "bf16" else (-23, 13)
    m, e = torch.frexp(amax)                      # amax = m 2^e, m in [0.5, 1)
    e = e.long() - 3 + (m > 0.75)
    return torch.where(amax > 0, e, lo).clamp(lo, hi)


def _levels(y):
    """Codes 0..7 of |y| (values 0 .5 1 1.5 2 3 4 6), nearest, ties to the even code."""
    return (y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0)


def _quantise(v, dt):
    """f32 or f64 [..., hd] -> code bytes [..., hd/2], scale bytes [..., hd/32]."""
    x = v.unflatten(-1, (-1, 32))
    e = _step(x.abs().amax(-1), dt)
    code = _levels(torch.ldexp(x.abs(), -e[..., None])) + 8 * torch.signbit(x).to(torch.uint8)
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _values(codes, scales, kind):
    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device, dtype=kind)
    v = torch.stack((lut[(codes & 15).long()], lut[(codes >> 4).long()]), -1).flatten(-2).unflatten(-1, (-1, 32))
    return torch.ldexp(v, scales.long()[..., None] - 127).flatten(-2)


def _held(c, pages, kind=torch.float32):
    """The values of a pool [npages][kv heads][page][hd]."""
    ps, hd = c["page"], c["hd"]
    if c["bits"] == 16:
        return pages.view(_TORCH[c["dt"]]).unflatten(-1, (ps, hd)).to(kind)
    return _values(pages[..., :ps * hd // 2].unflatten(-1, (ps, hd // 2)),
                   pages[..., ps * hd // 2:].unflatten(-1, (ps, hd // 32)), kind)


def _where(c, T):
    """For each row: its sequence, position, page and slot in the page."""
    rows = T["rows"].long()
    r = torch.arange(T["n"], device="cuda")
    s = torch.searchsorted(rows[1:], r, right=True)
    pos = T["len"].long()[s] - rows[s + 1] + r
    return s, pos, T["table"].long()[s, pos // c["page"]], pos % c["page"]


def _project(c, T, kind):
    """q, k, v of the rows in 32 (or 64) bits: normed and rotated, not yet rounded."""
    H, K, hd = c["heads"], c["kv_heads"], c["hd"]
    x = T["x"].unflatten(-1, (-1, hd)).to(kind)
    q, k, v = x[:, :H], x[:, H:H + K], x[:, H + K:]
    if c["norm"]:
        def norm(y, g):     # the sum of squares in 64 bits: a value next to a border of two codes keeps its side
            return (y * (1.0 / torch.sqrt((y.double() ** 2).mean(-1, keepdim=True) + 1e-6)).to(kind)) * g.to(kind)
        q, k = norm(q, T["gq"]), norm(k, T["gk"])
    if c["rope"]:
        pos = _where(c, T)[1]
        cs, sn = T["cos"][pos][:, None].to(kind), T["sin"][pos][:, None].to(kind)

        def turn(y):
            a, b = (y[..., 0::2], y[..., 1::2]) if c["rope"] == 1 else (y[..., :hd // 2], y[..., hd // 2:])
            a, b = a * cs - b * sn, b * cs + a * sn
            return torch.stack((a, b), -1).flatten(-2) if c["rope"] == 1 else torch.cat((a, b), -1)
        q, k = turn(q), turn(k)
    return q, k, v


def _plain_append(c, T):
    dt, ps, hd = _TORCH[c["dt"]], c["page"], c["hd"]
    q, k, v = _project(c, T, torch.float32)
    _, _, page, slot = _where(c, T)
    out = {"q": q.to(dt)}
    for name, y in (("kpages", k), ("vpages", v)):
        P = T[name]
        if c["bits"] == 16:
            P.view(dt).unflatten(-1, (ps, hd))[page, :, slot] = y.to(dt)
            out[name] = P.view(dt)
        else:
            codes, scales = _quantise(y, c["dt"])
            C, S = P[..., :ps * hd // 2].unflatten(-1, (ps, hd // 2)), P[..., ps * hd // 2:].unflatten(-1, (ps, hd // 32))
            C[page, :, slot], S[page, :, slot] = codes, scales
            out[name[0]] = _values(C[page, :, slot], S[page, :, slot], torch.float32).to(dt)
    return out


def _plain_attn(c, T):
    """The sequences padded to the longest: pages gathered, scores, softmax, sum."""
    H, K, hd, B, t, most = c["heads"], c["kv_heads"], c["hd"], c["batch"], T["t"], T["most"]
    rows = T["rows"].long()
    i = torch.arange(t, device="cuda")
    n = rows[1:] - rows[:-1]
    src = (rows[:-1, None] + i).clamp(max=T["n"] - 1)
    live = i < n[:, None]
    q = T["q"][src].float().view(B, t, K, H // K, hd).permute(0, 2, 3, 1, 4).reshape(B, K, -1, hd)
    used = T["table"][:, :-(-most // c["page"])].long().clamp(min=0)
    k, v = (_held(c, T[x][used]).transpose(1, 2).flatten(2, 3)[:, :, :most] for x in ("kpages", "vpages"))
    j = torch.arange(most, device="cuda")
    pos = T["len"].long()[:, None] - n[:, None] + i
    see = (j <= pos[..., None])[:, None, None]                                       # [B, 1, 1, t, most]
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(B, K, H // K, t, most)
    s = (s * hd ** -0.5).masked_fill(~see, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > -math.inf, m, 0.0))
    den = p.sum(-1, keepdim=True)
    v = v.masked_fill((j >= T["len"].long()[:, None])[:, None, :, None], 0.0)
    o = torch.matmul(p.view(B, K, -1, most), v).view(B, K, H // K, t, hd) / torch.where(den > 0, den, 1.0)
    return {"out": o.permute(0, 3, 1, 2, 4).reshape(B, t, H, hd)[live].to(_TORCH[c["dt"]])}


# ---- a program's side -------------------------------------------------------------

class _Buffer:
    """A device buffer of the framework, for torch too; freed with the last view of it."""

    def __init__(self, thvm, nbytes):
        self.buf = thvm.Buffer(nbytes)
        self.id = self.buf.id
        thvm.synchronize()                        # the zeros of a new buffer come before what torch writes
        self.__cuda_array_interface__ = dict(shape=(nbytes,), typestr="|u1", version=2,
                                             data=(thvm.lib().thvm_hip_buf_device_ptr(self.id), False))

    def __del__(self):
        self.buf.free()


class _Calls:
    """The buffers and the program texts that a server of these requests keeps."""

    def __init__(self, c, p, T):
        import thvm_amd as thvm
        thvm.init()
        self.thvm, self.bufs = thvm, {}
        n, H, K, hd, dt = p["n"], c["heads"], c["kv_heads"], c["hd"], _TORCH[c["dt"]]
        shape = dict(n=n, b=c["batch"], hkv=K, hd=hd, page=c["page"], maxpages=p["maxpages"], npages=p["npages"],
                     dt=_DT[c["dt"]], bits=c["bits"])
        ragged = any(r != p["t"] for r, _ in p["L"])
        if ragged:
            shape["ragged"] = 1
        rows = ["rows"] if ragged else []
        for name, v in T.items():
            if isinstance(v, torch.Tensor):
                self.torch(name, v.numel() * v.element_size()).copy_(v.contiguous().view(torch.uint8).flatten())
        pages = ["kpages", "vpages"]
        self.ops = []
        if c["op"] == "append":
            out = {"q": self.torch("q", n * H * hd * 2).view(dt).view(n, H, hd)}
            names = ["q"] + pages + ["x", "table", "len"] + rows + (["gq", "gk"] if c["norm"] else []) + \
                (["cos", "sin"] if c["rope"] else [])
            self.add("kv_append", names, (0, 1, 2), h=H, rope=c["rope"], norm=int(c["norm"]), eps=1e-6, **shape)
            if c["bits"] == 4:
                out.update({x: self.torch(x, n * K * hd * 2).view(dt).view(n, K, hd) for x in ("k", "v")})
                self.add("kv_read", ["k", "v"] + pages + ["table", "len"] + rows, (0, 1), **shape)
            else:
                out.update({x: self.torch(x, T[x].numel()).view(dt).view(p["npages"], K, -1) for x in pages})
        else:
            out = {"out": self.torch("out", n * H * hd * 2).view(dt).view(n, H, hd)}
            kw = dict(h=H, scale=hd ** -0.5, t=p["t"], **shape)
            self.torch("ws", max(16, thvm.attn_paged_ws(**kw)))
            self.add("attn_paged", ["out", "q"] + pages + ["table", "len"] + rows + ["ws"], (0,), **kw)
        self.out = out

    def torch(self, name, nbytes):
        if name not in self.bufs:
            self.bufs[name] = _Buffer(self.thvm, nbytes)
        return torch.as_tensor(self.bufs[name], device="cuda")

    def add(self, kernel, names, outs, **kw):
        text = " ".join("%s=%s" % (k, v.hex() if isinstance(v, float) else int(v)) for k, v in kw.items())
        self.ops.append((kernel, "thvm-builtin:%s %s" % (kernel, text), [self.bufs[x].id for x in names], outs))

    def run(self):
        for kernel, program, args, outs in self.ops:
            self.thvm.dispatch(kernel, program, args, outs=outs)
        return self.out


def prepare(case, seed):
    c = dict(case)
    p, T = _inputs(c, seed)
    state = {"case": c, "T": {**T, **p}}
    if own:
        state = {"case": c, "calls": _Calls(c, p, T)}
        torch.cuda.synchronize()
    return state


def run(state):
    if own:
        return state["calls"].run()
    c = state["case"]
    return _plain_append(c, state["T"]) if c["op"] == "append" else _plain_attn(c, state["T"])


# ---- the same in 64 bits -------------------------------------------------------------

def exact(case, seed):
    c = dict(case)
    p, T = _inputs(c, seed)
    H, K, hd, ps = c["heads"], c["kv_heads"], c["hd"], c["page"]
    f64 = torch.float64
    if c["op"] == "append":
        x, r0 = T["x"].to(f64).view(p["n"], H + 2 * K, hd), 0
        pools = {k: T[k].view(_TORCH[c["dt"]]).to(f64) for k in ("kpages", "vpages")} if c["bits"] == 16 else {}
        got = {"q": [], "k": [], "v": []}
        for s, (r, t) in enumerate(p["L"]):
            y, pos = x[r0:r0 + r].clone(), torch.arange(t - r, t, device="cuda")
            for part, gain in ((slice(0, H), "gq"), (slice(H, H + K), "gk")):
                z = y[:, part]
                if c["norm"]:
                    z = z * T[gain].to(f64) / ((z * z).sum(-1, keepdim=True) / hd + 1e-6).sqrt()
                if c["rope"]:   # as complex numbers, times e^(i angle) as the tables hold it
                    w = torch.complex(T["cos"][pos].to(f64), T["sin"][pos].to(f64))[:, None]
                    if c["rope"] == 1:
                        z = torch.view_as_real(torch.view_as_complex(z.contiguous().unflatten(-1, (-1, 2))) * w).flatten(-2)
                    else:
                        u = torch.complex(z[..., :hd // 2].contiguous(), z[..., hd // 2:].contiguous()) * w
                        z = torch.cat((u.real, u.imag), -1)
                y[:, part] = z
            page = T["table"][s].long()[pos // ps]
            for name, part in (("k", slice(H, H + K)), ("v", slice(H + K, None))):
                if c["bits"] == 16:
                    pools[name + "pages"].unflatten(-1, (ps, hd))[page, :, pos % ps] = y[:, part]
                else:
                    z = y[:, part].reshape(r, K, -1, 32)
                    lo, hi = (-126, 125) if c["dt"] == "bf16" else (-23, 13)
                    e = torch.ceil(torch.log2(z.abs().amax(-1, keepdim=True) / 6.0)).clamp(lo, hi)
                    w = z / 2.0 ** e
                    unit = 2.0 ** (torch.floor(torch.log2(w.abs().clamp(min=1.0))) - 1)   # spacing of the codes' values
                    got[name].append((torch.round(w / unit) * unit).clamp(-6, 6).mul(2.0 ** e).view(r, K, hd))
            got["q"].append(y[:, :H])
            r0 += r
        return {"q": torch.cat(got["q"]), **pools, **{k: torch.cat(got[k]) for k in ("k", "v") if got[k]}}
    outs, r0 = [], 0
    for s, (r, t) in enumerate(p["L"]):
        ids = T["table"][s, :-(-t // ps)].long()
        k, v = (_held(c, T[x][ids], f64).transpose(1, 2).reshape(-1, K, hd)[:t].transpose(0, 1).contiguous() for x in ("kpages", "vpages"))
        late = torch.arange(t, device="cuda") > torch.arange(t - r, t, device="cuda")[:, None]
        o = torch.empty(r, H, hd, device="cuda", dtype=f64)
        for h in range(H):
            a = T["q"][r0:r0 + r, h].to(f64) @ k[h // (H // K)].T.contiguous() / math.sqrt(hd)
            o[:, h] = torch.softmax(a.masked_fill(late, -math.inf), -1) @ v[h // (H // K)]
        outs.append(o)
        r0 += r
    return {"out": torch.cat(outs)}
