"""The 8-bit attention cache: head norms with the rotation, the store, the read back and the attention.

A numpy restatement keeps the cache's codes in natural order ([page, head, position, dim]) and packs them into
records by the documented byte order; everything is compared with float64.  Codes and scales have to be equal:
they are a function of f32 values that both sides round once from 64 bits.
"""
import ctypes as C

import numpy as np
import pytest

from blog_amd import qlin

BLOCK, RING = 32, 64
OK, UNSUP, SHAPE, NULL, ROWB, LIMIT, LAUNCH, ALIGN = range(8)
EPS = 1e-6
HEAD_DIMS = [64, 96, 128, 192, 256]


# ---- the restatement ---------------------------------------------------------------------------

def key_byte(t, d):
    return 1024 * (d // 32) + 256 * (d // 8 % 4) + 16 * (t % 16) + 8 * (t // 16) + d % 8


def value_byte(t, d, head_dim):
    w = d // 4 + t % 2 * (head_dim // 4)
    return 1024 * (w // 16) + 256 * (t // 4 % 4) + 16 * (w % 16) + 8 * (t // 16) + 4 * (t // 2 % 2) + d % 4


def byte_maps(d):
    t, e = np.meshgrid(np.arange(BLOCK), np.arange(d), indexing="ij")
    return key_byte(t, e), 32 * d + value_byte(t, e, d)


def pack(kc, vc, scales, spare=0):
    """Codes [pages, heads, 32, d] and scales [pages, heads, 2] to pages [pages, heads, 64 d + 16]."""
    p, h, _, d = kc.shape
    out = np.full((p, h, 64 * d + 16), spare, np.uint8)
    km, vm = byte_maps(d)
    out[:, :, km] = kc.view(np.uint8)
    out[:, :, vm] = vc.view(np.uint8)
    out[:, :, 64 * d:64 * d + 8] = np.ascontiguousarray(scales.astype(np.float32)).view(np.uint8).reshape(p, h, 8)
    return out


def unpack(pages, d):
    km, vm = byte_maps(d)
    scales = np.ascontiguousarray(pages[:, :, 64 * d:64 * d + 8]).view(np.float32)
    return pages[:, :, km].view(np.int8), pages[:, :, vm].view(np.int8), scales


def quantize(x):
    """x [32, d] f32: codes and the scale, in f32 as documented."""
    top = np.abs(x).max()
    if not np.isfinite(top):
        return np.zeros(x.shape, np.int8), np.float32(np.nan)
    s = np.float32(top) * (np.float32(1) / np.float32(127))
    if s == 0:
        return np.zeros(x.shape, np.int8), s
    return np.clip(np.rint(x / s), -127, 127).astype(np.int8), s


def table64(n, rd, theta):
    i = np.arange(rd // 2)
    a = np.arange(n)[:, None] * theta ** (-2.0 * i / max(rd, 1))
    return np.concatenate([np.cos(a), np.sin(a)], 1)


def norm_rope(x, w, table, pos, rd, pairing, eps=EPS):
    """x [rows, heads, d] float64 at positions pos; w [d] or None; table [n, rd] as the f32 values."""
    if w is not None:
        x = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * w
    x = x.copy()
    if rd:
        row = table[np.clip(pos, 0, len(table) - 1)].astype(np.float64)
        c, s = row[:, None, :rd // 2], row[:, None, rd // 2:]
        a, b = (slice(0, rd, 2), slice(1, rd, 2)) if pairing else (slice(0, rd // 2), slice(rd // 2, rd))
        u, v = x[..., a].copy(), x[..., b].copy()
        x[..., a], x[..., b] = u * c - v * s, v * c + u * s
    return x


class Cache:
    """The documented behaviour of qlin_kv8_cache, position by position."""

    def __init__(self, n_seqs, per, kv, d, table=None, n_pages=None):
        self.n, self.per, self.kv, self.d = n_seqs, per, kv, d
        self.table = np.arange(n_seqs * per).reshape(n_seqs, per) if table is None else table
        self.n_pages = n_pages or n_seqs * per
        self.kc = np.zeros((self.n_pages, kv, BLOCK, d), np.int8)
        self.vc = np.zeros_like(self.kc)
        self.scales = np.zeros((self.n_pages, kv, 2), np.float32)
        self.ring = np.zeros((n_seqs, kv, 2, RING, d), np.float32)
        self.history = [dict() for _ in range(n_seqs)]  # position -> (k, v) f32 [kv, d], as last stored

    def page(self, s, b):
        p = self.table[s, b]
        return p if 0 <= p < self.n_pages else None

    def store(self, s, start, k, v):
        """k, v [rows, kv, d] f32 at start .."""
        cap = self.per * BLOCK
        start = min(start, cap)
        length = max(0, min(start + len(k), cap))
        fresh = [p for p in range(max(start, 0), length)]
        if not fresh:
            return
        ring = self.ring[s].copy()  # positions before the call's own are the ring's
        for p in range(fresh[0] // BLOCK * BLOCK, fresh[0]):
            if p in self.history[s]:  # (else a start past the last end: whatever is there)
                assert all(np.array_equal(ring[:, j, p % RING], self.history[s][p][j]) for j in range(2))
            else:
                self.history[s][p] = (ring[:, 0, p % RING], ring[:, 1, p % RING])
        for p in fresh:
            self.history[s][p] = (k[p - start], v[p - start])
        last = (length - 1) // BLOCK
        for b in range(fresh[0] // BLOCK, last + 1):
            if b >= last - 1:
                for p in fresh:
                    if p // BLOCK == b:
                        self.ring[s, :, 0, p % RING], self.ring[s, :, 1, p % RING] = self.history[s][p]
            page = self.page(s, b)
            if (b + 1) * BLOCK > length or page is None:
                continue
            for h in range(self.kv):
                for j, codes in ((0, self.kc), (1, self.vc)):
                    x = np.stack([self.history[s][p][j][h] for p in range(b * BLOCK, (b + 1) * BLOCK)])
                    codes[page, h], self.scales[page, h, j] = quantize(x)

    def values(self, s, length):
        """K, V [length, kv, d] float64 that the cache stands for, and which positions are seen."""
        length = max(0, min(length, self.per * BLOCK))
        out, there = np.zeros((2, length, self.kv, self.d)), np.zeros(length, bool)
        for p in range(length):
            b, page = p // BLOCK, self.page(s, p // BLOCK)
            if page is None:
                continue
            there[p] = True
            if (b + 1) * BLOCK <= length:
                for j, codes in ((0, self.kc), (1, self.vc)):
                    out[j, p] = codes[page, :, p % BLOCK].astype(np.float64) * self.scales[page, :, j, None].astype(np.float64)
            else:
                out[0, p], out[1, p] = self.ring[s, :, 0, p % RING], self.ring[s, :, 1, p % RING]
        return out[0], out[1], there


def attend(q, k, v, there, start, scale):
    """q [rows, heads, d]; k, v [length, kv, d]; float64.  Also, for the tolerance, the largest sum of a score's
    magnitudes and the largest value."""
    rows, heads, d = q.shape
    out, big = np.zeros((rows, heads, d)), 0.0
    for r in range(rows):
        see = np.flatnonzero(there & (np.arange(len(k)) <= start + r))
        if not len(see):
            continue
        for h in range(heads):
            g = h // (heads // k.shape[1])
            s = k[see, g] @ q[r, h] * scale
            big = max(big, np.nanmax(np.abs(k[see, g]) @ np.abs(q[r, h])) * abs(scale))
            with np.errstate(invalid="ignore"):
                e = np.exp(s - s.max())
                out[r, h] = (e / e.sum()) @ v[see, g]
    return out, big


def attend_tolerance(big, v):
    """A score s log2(e) of magnitudes that sum to `big` is off by: q's factor (one rounding), the products' sum and its
    scale (a chain of head_dim / 32 MFMA steps, each off by at most two roundings of the sum so far, 16 of them taken
    at head_dim 256, and the codes' scale), the subtraction of the maximum; a probability by that times ln 2 and
    2^-22 (v_exp_f32, its part in the sums); the output by twice the probabilities' relative error (numerator and
    denominator) and a rounding for each of the joins (blocks of a wave, waves, splits: fewer than 64)."""
    step = 2.0 ** -24
    score = (16 + 4) * step * big * 1.4427
    return (2 * (score * 0.6932 + 2.0 ** -22) + 64 * step) * max(1e-30, np.nanmax(np.abs(v)) if v.size else 0.0)


# ---- CPU ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("d", HEAD_DIMS)
def test_records_hold_every_code_once(d):
    km, vm = byte_maps(d)
    assert sorted(np.concatenate([km.ravel(), vm.ravel()])) == list(range(64 * d))
    rng = np.random.default_rng(d)
    kc, vc = (rng.integers(-127, 128, (2, 3, BLOCK, d)).astype(np.int8) for _ in range(2))
    s = rng.random((2, 3, 2)).astype(np.float32)
    for a, b in zip(unpack(pack(kc, vc, s), d), (kc, vc, s)):
        assert np.array_equal(a, b)
    assert qlin.kv8_record_bytes(d) == 64 * d + 16


def test_restatement_of_the_norm_and_the_turn():
    """Against a loop over pairs: x w / rms, then (a + i b) e^(i angle)."""
    rng = np.random.default_rng(3)
    x, w = rng.standard_normal((4, 2, 32)), rng.standard_normal(32)
    pos, rd, theta = np.array([0, 3, 500, 70000]), 16, 1e4
    t = table64(70001, rd, theta)
    for pairing in (0, 1):
        y = norm_rope(x, w, t, pos, rd, pairing)
        for r in range(4):
            for h in range(2):
                z = x[r, h] * w / np.sqrt((x[r, h] ** 2).sum() / 32 + EPS)
                for i in range(rd // 2):
                    a, b = (2 * i, 2 * i + 1) if pairing else (i, i + rd // 2)
                    turned = (z[a] + 1j * z[b]) * np.exp(1j * pos[r] * theta ** (-2 * i / rd))
                    z[a], z[b] = turned.real, turned.imag
                assert np.allclose(y[r, h], z, rtol=1e-12, atol=1e-12)


FAKE = 0x10000


def _how(**kw):
    a = dict(q_norm=FAKE, k_norm=FAKE, norm_type=0, eps=EPS, one_plus=0, table=FAKE, table_len=100, rotary_dim=64, pairing=0)
    a.update(kw)
    return qlin.QkRopeArgs(*a.values())


def _cache(**kw):
    a = dict(pages=FAKE, recent=FAKE, block_table=FAKE, n_pages=8, n_seqs=2, blocks_per_seq=4, kv_heads=2, head_dim=64)
    a.update(kw)
    return qlin.Kv8CacheArgs(*a.values())


BAD_HOW = [(dict(norm_type=2), SHAPE), (dict(rotary_dim=72), SHAPE), (dict(rotary_dim=-8), SHAPE), (dict(rotary_dim=12), SHAPE),
           (dict(pairing=2), SHAPE), (dict(table_len=0), SHAPE), (dict(table=None), NULL), (dict(q_norm=FAKE + 1), ALIGN),
           (dict(k_norm=FAKE + 1), ALIGN), (dict(table=FAKE + 2), ALIGN)]
BAD_CACHE = [(dict(kv_heads=0), SHAPE), (dict(n_seqs=-1), SHAPE), (dict(blocks_per_seq=0), SHAPE), (dict(n_pages=0), SHAPE),
             (dict(head_dim=0), SHAPE), (dict(head_dim=80), LIMIT), (dict(head_dim=512), LIMIT), (dict(blocks_per_seq=32769), LIMIT),
             (dict(block_table=None, n_pages=7), SHAPE), (dict(pages=None), NULL), (dict(recent=None), NULL),
             (dict(pages=FAKE + 8), ALIGN), (dict(recent=FAKE + 4), ALIGN), (dict(block_table=FAKE + 2), ALIGN)]


def test_rope_table_validation():
    run = lambda t=FAKE, n=10, rd=64, theta=1e4: qlin.status("qlin_launch_rope_table", t, n, rd, theta)
    assert run(n=-1) == SHAPE and run(rd=63) == SHAPE and run(rd=-2) == SHAPE
    assert run(theta=0.0) == SHAPE and run(theta=float("nan")) == SHAPE and run(theta=float("inf")) == SHAPE
    assert run(n=(1 << 20) + 1) == LIMIT and run(rd=258) == LIMIT
    assert run(t=0) == NULL and run(t=FAKE + 2) == ALIGN
    assert run(n=0, t=0) == OK and run(rd=0, t=0) == OK


def test_norm_rope_store_validation():
    def run(how=None, q=FAKE, qs=256, k=FAKE, ks=128, v=FAKE, vs=128, qo=FAKE + 4096, kc=FAKE, vc=FAKE, rows=1, nh=4, kv=2, hd=64,
            ms=100, pos=FAKE):
        h = _how() if how is None else how
        return qlin.status("qlin_launch_qk_norm_rope_store_kv", C.addressof(h) if h else None, q, qs, k, ks, v, vs, qo, kc, vc,
                           rows, nh, kv, hd, ms, pos)
    for kw, rc in BAD_HOW:
        assert run(how=_how(**kw)) == rc, kw
    assert run(how=False) == NULL
    assert run(nh=5) == SHAPE and run(kv=0) == SHAPE and run(hd=60) == SHAPE and run(rows=-1) == SHAPE and run(ms=0) == SHAPE
    assert run(hd=264, qs=9999, ks=999, vs=999) == LIMIT and run(ms=(1 << 20) + 1) == LIMIT
    assert run(qs=255) == SHAPE and run(ks=127) == SHAPE and run(vs=127) == SHAPE
    assert run(q=FAKE, qo=FAKE, qs=300) == SHAPE  # in place needs packed queries
    for name in ("q", "k", "v", "qo", "kc", "vc", "pos"):
        assert run(**{name: 0}) == NULL, name
        assert run(**{name: FAKE + 2}) == ALIGN, name
    assert run(rows=0, q=0, k=0, v=0, qo=0, kc=0, vc=0, pos=0) == OK
    assert run(rows=0, how=_how(table=None, rotary_dim=0, table_len=0, q_norm=None, k_norm=None)) == OK


def test_store_kv8_validation():
    def run(how=None, cache=None, q=FAKE, qs=256, k=FAKE, ks=128, v=FAKE, vs=128, qo=FAKE + 4096, rows=1, nh=4, pos=FAKE, nr=None):
        h, c = _how() if how is None else how, _cache() if cache is None else cache
        return qlin.status("qlin_launch_qk_norm_rope_store_kv8", C.addressof(h) if h else None, C.addressof(c) if c else None, q,
                           qs, k, ks, v, vs, qo, rows, nh, pos, nr)
    for kw, rc in BAD_HOW:
        assert run(how=_how(**kw)) == rc, kw
    for kw, rc in BAD_CACHE:
        assert run(cache=_cache(**kw)) == rc, kw
    assert run(how=False) == NULL and run(cache=False) == NULL
    assert run(nh=3) == SHAPE and run(rows=-1) == SHAPE and run(rows=(1 << 20) + 1) == LIMIT
    assert run(qs=255) == SHAPE and run(ks=127) == SHAPE and run(vs=127) == SHAPE and run(q=FAKE, qo=FAKE, qs=300) == SHAPE
    for name in ("q", "k", "v", "qo", "pos"):
        assert run(**{name: 0}) == NULL, name
        assert run(**{name: FAKE + 2}) == ALIGN, name
    assert run(nr=FAKE + 1) == ALIGN
    assert run(rows=0, q=0, k=0, v=0, qo=0, pos=0) == OK
    assert run(cache=_cache(n_seqs=0), q=0, k=0, v=0, qo=0, pos=0) == OK


def test_read_and_attend_validation():
    def read(cache=None, first=FAKE, lens=FAKE, count=3, ko=FAKE, vo=FAKE):
        c = _cache() if cache is None else cache
        return qlin.status("qlin_launch_kv8_read", C.addressof(c) if c else None, first, lens, count, ko, vo)

    def att(cache=None, q=FAKE, out=FAKE, rows=1, nh=4, pos=FAKE, nr=None, scale=0.1, ws=FAKE, nws=1 << 40):
        c = _cache() if cache is None else cache
        return qlin.status("qlin_launch_attend_kv8", C.addressof(c) if c else None, q, out, rows, nh, pos, nr, scale, ws, nws)
    for run in (read, att):
        for kw, rc in BAD_CACHE:
            assert run(cache=_cache(**kw)) == rc, kw
        assert run(cache=False) == NULL
    for name in ("first", "lens", "ko", "vo"):
        assert read(**{name: 0}) == NULL, name
        assert read(**{name: FAKE + 2}) == ALIGN, name
    assert read(count=-1) == SHAPE and read(count=0, first=0, lens=0, ko=0, vo=0) == OK
    assert att(nh=3) == SHAPE and att(rows=-1) == SHAPE and att(scale=float("nan")) == SHAPE and att(scale=float("inf")) == SHAPE
    assert att(rows=(1 << 20) + 1) == LIMIT
    for name in ("q", "out", "pos"):
        assert att(**{name: 0}) == NULL, name
    assert att(q=FAKE + 4) == ALIGN and att(out=FAKE + 8) == ALIGN and att(pos=FAKE + 1) == ALIGN and att(nr=FAKE + 1) == ALIGN
    assert att(ws=FAKE + 8) == ALIGN
    assert att(rows=0, q=0, out=0, pos=0, ws=0, nws=0) == OK
    # a cache long enough for splits needs its workspace
    big = _cache(blocks_per_seq=1000, n_pages=2000)
    need = qlin.attend_kv8_workspace_bytes(2, 1, 4, 2, 64, 1000)
    assert need > 0 and att(cache=big, ws=0, nws=0) == NULL and att(cache=big, nws=need - 1) == LIMIT
    assert qlin.attend_kv8_workspace_bytes(0, 1, 4, 2, 64, 1000) == 0
    assert qlin.attend_kv8_workspace_bytes(2, 1, 5, 2, 64, 1000) == 0


def test_python_cache_checks_its_tensors():
    import torch
    c = qlin.Kv8Cache.empty(torch, 2, 3, 64, 100, device="cpu")
    assert (c.blocks_per_seq, c.n_seqs, c.kv_heads, c.head_dim) == (4, 2, 3, 64)
    with pytest.raises(ValueError):
        qlin.Kv8Cache(c.pages[:, :, :-1].contiguous(), c.recent, None, 4)
    with pytest.raises(ValueError):
        qlin.Kv8Cache(c.pages, c.recent[:, :, :, :32].contiguous(), None, 4)
    with pytest.raises(ValueError):
        qlin.Kv8Cache(c.pages, c.recent, torch.zeros(3, 4, dtype=torch.int32))
    with pytest.raises(ValueError):
        qlin.Kv8Cache(c.pages, c.recent, torch.zeros(4, 2, dtype=torch.int32).t())


def test_python_tensors_of_other_types():
    import torch
    c = qlin.Kv8Cache.empty(torch, 2, 3, 64, 100, device="cpu")
    with pytest.raises(ValueError):
        qlin.Kv8Cache(c.pages, c.recent, torch.zeros(2, 4, dtype=torch.int64))
    with pytest.raises(ValueError):
        qlin.Kv8Cache(c.pages.to(torch.int16), c.recent, None, 4)
    with pytest.raises(ValueError):
        qlin.Kv8Cache(c.pages, c.recent.half(), None, 4)
    table, w = torch.zeros(100, 64), torch.ones(64, dtype=torch.bfloat16)
    assert qlin.QkRope(w, w, 0, 1e-6, 0, table, 64).args.table_len == 100
    for bad in (dict(table=table.half()), dict(table=torch.zeros(100, 32)), dict(table=torch.zeros(64, 100).t()),
                dict(q_norm=w.float()), dict(k_norm=torch.ones(128, dtype=torch.float16)[::2])):
        a = {**dict(q_norm=w, k_norm=w, norm_type=0, eps=1e-6, one_plus=0, table=table, rotary_dim=64), **bad}
        with pytest.raises(ValueError):
            qlin.QkRope(**a)
    with pytest.raises(ValueError):
        qlin.rope_table(torch.zeros(64, 100).t(), 1e4)


# ---- GPU ---------------------------------------------------------------------------------------

def _gpu():
    import torch
    from gpu_util import bind_stream
    assert torch.cuda.is_available(), "GPU tests need the MI355X"
    bind_stream()
    return torch


def bits_of(w, norm_type):
    """Norm weights as 16-bit patterns, and their values."""
    if norm_type == 0:
        b = (w.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)
        return b, (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    h = w.astype(np.float16)
    return h.view(np.uint16), h.astype(np.float64)


@pytest.mark.gpu
@pytest.mark.parametrize("n,rd,theta", [(1, 2, 1e4), (257, 64, 1e6), (40000, 128, 5e5), (1000, 256, 1e7)])
def test_rope_table(n, rd, theta):
    torch = _gpu()
    from gpu_util import banner, empty_f32, host
    banner(f"rope_table {n} {rd}")
    t = empty_f32(n, rd)
    qlin.rope_table(t, theta)
    # half an f32 step of a value up to 1, and the angle's own error in 64 bits (n * 2^-52 of pow and product)
    assert np.abs(host(t) - table64(n, rd, np.float32(theta).astype(np.float64))).max() <= 2.0 ** -25 + n * 2.0 ** -50


@pytest.mark.gpu
@pytest.mark.parametrize("rows,heads,kv,d,rd,pairing,norm_type,one_plus,normed,start", [
    (1, 14, 2, 64, 64, 0, 0, 0, True, 37), (33, 6, 3, 128, 128, 0, 1, 0, True, 100), (5, 4, 4, 256, 64, 1, 0, 1, True, 0),
    (3, 7, 1, 96, 96, 1, 1, 1, True, 60), (70, 2, 2, 40, 16, 0, 0, 0, True, 29000), (2, 3, 1, 8, 8, 1, 0, 0, True, 3),
    (9, 8, 2, 16, 0, 0, 0, 0, True, 5), (4, 4, 2, 200, 200, 0, 0, 0, False, 11), (1, 4, 2, 24, 0, 0, 0, 0, False, 1)])
def test_norm_rope_store_f32_cache(rows, heads, kv, d, rd, pairing, norm_type, one_plus, normed, start):
    torch = _gpu()
    from gpu_util import banner, dev, empty_f32, host
    rng = np.random.default_rng(rows * d + rd)
    banner(f"qk_norm_rope_store_kv rows={rows} heads={heads}/{kv} d={d} rd={rd}")
    ms = start + rows + 3
    width = (heads + 2 * kv) * d + 5  # heads of a wider row: 4-byte alignment only
    x = (rng.standard_normal((rows, width)) * 10 ** rng.uniform(-2, 2, (rows, 1))).astype(np.float32)
    wq, vq = bits_of(rng.standard_normal(d) * 0.5 + 1, norm_type)
    wk, vk = bits_of(rng.standard_normal(d) * 0.5 + 1, norm_type)
    vq, vk = (vq + one_plus, vk + one_plus) if normed else (None, None)
    table = table64(ms, rd, 1e6).astype(np.float32)
    xd = dev(x)
    how = qlin.QkRope(dev(wq) if normed else None, dev(wk) if normed else None, norm_type, EPS, one_plus, dev(table) if rd else None, rd, pairing)
    q_out, kc, vc = empty_f32(rows, heads, d), empty_f32(ms, kv, d), empty_f32(ms, kv, d)
    pos = torch.tensor([start], dtype=torch.int32, device="cuda")
    a = xd.data_ptr() + 4 * 3
    qlin.qk_norm_rope_store_kv(how, a, width, a + 4 * heads * d, width, a + 4 * (heads + kv) * d, width, q_out, kc, vc, rows,
                               heads, kv, d, ms, pos)
    body = x[:, 3:3 + (heads + 2 * kv) * d].astype(np.float64).reshape(rows, heads + 2 * kv, d)
    p = start + np.arange(rows)
    q = norm_rope(body[:, :heads], vq, table, p, rd, pairing)
    k = norm_rope(body[:, heads:heads + kv], vk, table, p, rd, pairing)
    v = body[:, heads + kv:].astype(np.float32)
    # one rounding of a 64-bit result (whose own error is far below it)
    assert np.abs(host(q_out) - q).max() <= np.abs(q).max() * 2.0 ** -24
    assert (np.abs(host(q_out) - q) <= np.abs(q) * 2.0 ** -24 * 1.01 + np.abs(q).max() * 2.0 ** -50).all()
    kh, vh = host(kc), host(vc)
    assert (np.abs(kh[p] - k) <= np.abs(k) * 2.0 ** -24 * 1.01 + np.abs(k).max() * 2.0 ** -50).all()
    assert np.array_equal(vh[p], v)
    others = np.setdiff1d(np.arange(ms), p)
    assert np.isnan(kh[others]).all() and np.isnan(vh[others]).all()


@pytest.mark.gpu
def test_norm_rope_in_place_and_clamped_positions():
    """Queries in place; positions outside the cache clamped as qlin_launch_rope_store_kv clamps them; the norm of a zero
    head is zero, that of one with an infinity not a number."""
    torch = _gpu()
    from gpu_util import banner, dev, empty_f32, host
    heads, kv, d, ms = 4, 2, 64, 10
    rng = np.random.default_rng(2)
    table = table64(ms, d, 1e4).astype(np.float32)
    w, vw = bits_of(np.ones(d), 0)
    for start, at in ((-7, 0), (25, 9), (-2 ** 31, 0), (2 ** 31 - 1, 9)):
        banner(f"in place, start={start}")
        x = rng.standard_normal((heads + 2 * kv, d)).astype(np.float32)
        x[1] = 0
        x[2, 5] = np.inf
        q = dev(x[:heads])
        kc, vc = empty_f32(ms, kv, d), empty_f32(ms, kv, d)
        qlin.qk_norm_rope_store_kv(qlin.QkRope(dev(w), dev(w), 0, EPS, 0, dev(table), d), q, heads * d, dev(x[heads:heads + kv]), kv * d,
                                   dev(x[heads + kv:]), kv * d, q, kc, vc, 1, heads, kv, d, ms,
                                   torch.tensor([start], dtype=torch.int32, device="cuda"))
        with np.errstate(invalid="ignore"):
            ref = norm_rope(x[None].astype(np.float64), vw, table, np.array([at]), d, 0)[0]
        got = host(q)
        assert np.isnan(got[2]).any() and (got[1] == 0).all()
        for h in (0, 3):
            assert np.abs(got[h] - ref[h]).max() <= np.abs(ref[h]).max() * 2.0 ** -23
        assert np.abs(host(kc)[at] - ref[heads:heads + kv]).max() <= np.abs(ref[heads:heads + kv]).max() * 2.0 ** -23
        assert np.isnan(host(kc)[[p for p in range(ms) if p != at]]).all()


def _device_cache(torch, ref, paged):
    from gpu_util import dev
    pages = dev(pack(ref.kc, ref.vc, ref.scales, spare=0xA5))
    recent = dev(ref.ring)
    return qlin.Kv8Cache(pages, recent, dev(ref.table.astype(np.int32)) if paged else None, ref.per)


def _check_cache(ref, cache):
    from gpu_util import host
    pages = host(cache.pages)
    kc, vc, scales = unpack(pages, ref.d)
    assert np.array_equal(scales, ref.scales, equal_nan=True)
    assert np.array_equal(kc, ref.kc) and np.array_equal(vc, ref.vc)
    assert (pages[:, :, 64 * ref.d + 8:] == 0xA5).all()
    ring = host(cache.recent)
    assert np.array_equal(ring[:, :, 1], ref.ring[:, :, 1], equal_nan=True)
    # Both sides round a key once to f32, from 64-bit results that differ by a few 2^-52 of it: the same value, but for
    # the rare one (about 1 in 10^8) whose 64-bit results lie on two sides of a border, which is one f32 step off.
    got, want = ring[:, :, 0], ref.ring[:, :, 0]
    assert np.array_equal(np.isnan(got), np.isnan(want))
    off = ~np.isnan(want) & (got != want)
    assert off.sum() <= 2 and (np.abs(got - want)[off] <= np.spacing(np.abs(want[off]))).all(), (off.sum(), got[off], want[off])


def _store(torch, ref, cache, rng, starts, rows, counts, heads, how_args, poison=None):
    """One store of random rows into both; returns nothing, checks the queries and the cache."""
    from gpu_util import dev, empty_f32, host
    n, kv, d = ref.n, ref.kv, ref.d
    w, vw, norm_type, one_plus, table, rd, pairing = how_args
    how = qlin.QkRope(*([dev(w), dev(w)] if w is not None else [None, None]), norm_type, EPS, one_plus, dev(table) if rd else None, rd, pairing)
    width = (heads + 2 * kv) * d
    x = (rng.standard_normal((n, rows, heads + 2 * kv, d)) * 10 ** rng.uniform(-1, 1, (1, 1, heads + 2 * kv, 1))).astype(np.float32)
    if poison is not None:
        poison(x)
    xd = dev(x)
    a = xd.data_ptr()
    q_out = empty_f32(n, rows, heads, d)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    qlin.qk_norm_rope_store_kv8(how, cache, a, width, a + 4 * heads * d, width, a + 4 * (heads + kv) * d, width, q_out, rows, heads,
                                i32(starts), None if counts is None else i32(counts))
    got = host(q_out)
    for s in range(n):
        c = rows if counts is None else max(0, min(counts[s], rows))
        with np.errstate(invalid="ignore"):
            turned = norm_rope(x[s, :c, :heads + kv].astype(np.float64), vw, table, starts[s] + np.arange(c), rd, pairing)
        q = turned[:, :heads]
        assert (np.abs(got[s, :c] - q) <= np.abs(q) * 2.0 ** -24 * 1.01 + 1e-30 + np.abs(q).max(initial=0) * 2.0 ** -50).all()
        assert np.isnan(got[s, c:]).all()  # left as they were
        ref.store(s, starts[s], turned[:, heads:].astype(np.float32), x[s, :c, heads + kv:])
    _check_cache(ref, cache)


def _norm_args(rng, d, rd, cap, normed=True, norm_type=0, one_plus=0, pairing=0):
    w, vw = bits_of(rng.standard_normal(d) * 0.5 + 1, norm_type)
    return (w if normed else None, vw + one_plus if normed else None, norm_type, one_plus,
            table64(cap, rd, 1e5).astype(np.float32), rd, pairing)


@pytest.mark.gpu
@pytest.mark.parametrize("d,heads,kv,rd,pairing,normed,norm_type,one_plus", [
    (64, 6, 2, 64, 0, True, 0, 0), (96, 3, 3, 48, 1, True, 1, 1), (128, 8, 2, 128, 0, True, 1, 0), (192, 2, 1, 192, 1, False, 0, 0),
    (256, 2, 2, 128, 0, True, 0, 1), (128, 1, 1, 0, 0, False, 0, 0)])
def test_store_in_pieces(d, heads, kv, rd, pairing, normed, norm_type, one_plus):
    """Prompts, single tokens, chunks that end and begin inside blocks, rejected drafts: the cache as a whole after each
    call, to the last byte."""
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(d + heads)
    ref = Cache(1, 10, kv, d)
    cache = _device_cache(torch, ref, paged=False)
    args = _norm_args(rng, d, rd, 320, normed, norm_type, one_plus, pairing)
    # start, rows: a chunk of 150 from 20 has a last block that takes the first one's ring rows; (-4, +) goes back
    for start, rows in ((0, 20), (20, 150), (170, 1), (171, 4), (173, 1), (174, 1), (175, 16), (191, 1), (192, 1), (193, 8),
                        (170, 31), (201, 64), (265, 33), (298, 22)):
        banner(f"store d={d} start={start} rows={rows}")
        _store(torch, ref, cache, rng, [start], rows, None, heads, args)


@pytest.mark.gpu
def test_store_token_by_token_gives_the_prompts_bytes():
    torch = _gpu()
    from gpu_util import banner, dev, empty_f32, host
    rng = np.random.default_rng(9)
    heads, kv, d, n = 4, 2, 128, 77
    x = dev(rng.standard_normal((n, (heads + 2 * kv) * d)).astype(np.float32))
    w, _, _, _, table, rd, _ = _norm_args(rng, d, d, 96)
    how = qlin.QkRope(dev(w), dev(w), 0, EPS, 0, dev(table), rd)
    width, got = (heads + 2 * kv) * d, []
    for step in (n, 1, 7):
        banner(f"store in steps of {step}")
        cache = qlin.Kv8Cache.empty(torch, 1, kv, d, 96)
        q = empty_f32(n, heads, d)
        for i in range(0, n, step):
            rows = min(step, n - i)
            a = x.data_ptr() + 4 * width * i
            qlin.qk_norm_rope_store_kv8(how, cache, a, width, a + 4 * heads * d, width, a + 4 * (heads + kv) * d, width, q[i:], rows,
                                        heads, torch.tensor([i], dtype=torch.int32, device="cuda"))
        got.append((host(cache.pages), host(q), host(cache.recent)[:, :, :, [p % 64 for p in range(32, n)]]))
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert np.array_equal(a, b)


@pytest.mark.gpu
def test_store_of_another_sequence_over_a_longer_one():
    """From position 0, and from a block's first position, after more positions were stored."""
    torch = _gpu()
    rng = np.random.default_rng(77)
    ref, heads = Cache(2, 7, 2, 64), 4
    cache = _device_cache(torch, ref, paged=False)
    how = _norm_args(rng, 64, 64, 7 * BLOCK)
    for starts, rows in (([0, 0], 203), ([0, 32], 7), ([7, 39], 1), ([8, 40], 90), ([0, 96], 64), ([64, 160], 5)):
        _store(torch, ref, cache, rng, starts, rows, None, heads, how)
        _check_cache(ref, cache)
        q = rng.standard_normal((2, rows, heads, 64)).astype(np.float32)
        _check_attend(torch, ref, cache, q, starts, None, heads, 0.125)


@pytest.mark.gpu
def test_store_of_a_padded_batch():
    """Sequences with rows of their own: none, all, some; a table in no order with a page that is not there; starts
    outside the cache."""
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(4)
    n, per, kv, d, heads = 7, 3, 2, 64, 4
    table = rng.permutation(n * per + 5)[:n * per].reshape(n, per)
    table[1, 1] = -1
    table[2, 0] = 1 << 30
    ref = Cache(n, per, kv, d, table, n * per + 5)
    cache = _device_cache(torch, ref, paged=True)
    args = _norm_args(rng, d, d, 96)
    for starts, rows, counts in (([0] * n, 40, [40, 39, 33, 0, -5, 99, 1]),
                                 ([40, 39, 33, 0, 0, 40, 1], 1, None),
                                 ([41, 40, 34, 1, 1, 41, 2], 60, [60, 24, 30, 60, 31, 55, 0]),
                                 ([96, 200, -3, -70, 2 ** 31 - 1, -2 ** 31, 90], 9, None)):
        banner(f"padded batch rows={rows}")
        _store(torch, ref, cache, rng, starts, rows, counts, heads, args)


@pytest.mark.gpu
def test_store_of_values_that_are_odd():
    """Blocks of zeros, of the smallest subnormals, with an infinity, with a NaN: the documented scales and codes."""
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(5)
    kv, d, heads = 1, 64, 1
    ref = Cache(1, 6, kv, d)
    cache = _device_cache(torch, ref, paged=False)
    args = _norm_args(rng, d, 0, 192, normed=False)

    def poison(x):
        x[0, 0:32, 1:] = 0
        x[0, 32:64, 1:] = (rng.integers(-70, 71, (32, 2, d)) * 1.401298464324817e-45).astype(np.float32)
        x[0, 70, 1, 3] = np.inf
        x[0, 75, 2, 3] = np.nan
        x[0, 100, 1, 5] = -np.inf
        x[0, 130:140, 2] = 3e38
    banner("store of odd values")
    _store(torch, ref, cache, rng, [0], 170, None, heads, args, poison)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 192])
def test_read_back(d):
    torch = _gpu()
    from gpu_util import banner, dev, empty_f32, host
    rng = np.random.default_rng(d)
    n, per, kv = 3, 4, 2
    table = rng.permutation(20)[:n * per].reshape(n, per)
    table[1, 0] = -1
    ref = _filled(rng, n, per, kv, d, table, 20)
    cache = _device_cache(torch, ref, paged=True)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    for first, lens, count in (([0, 0, 0], [128, 70, 0], 128), ([31, 5, 64], [90, 64, 65], 33), ([-3, 100, -2 ** 31], [500, 128, -1], 50)):
        banner(f"read d={d} first={first}")
        k, v = empty_f32(n, count, kv, d), empty_f32(n, count, kv, d)
        qlin.kv8_read(cache, i32(first), i32(lens), count, k, v)
        k, v = host(k), host(v)
        for s in range(n):
            kr, vr, there = ref.values(s, lens[s])
            for r in range(count):
                p = first[s] + r
                if 0 <= p < len(there) and there[p]:
                    assert np.array_equal(k[s, r], kr[p].astype(np.float32)) and np.array_equal(v[s, r], vr[p].astype(np.float32))
                else:
                    assert np.isnan(k[s, r]).all() and np.isnan(v[s, r]).all()


def _filled(rng, n, per, kv, d, table=None, n_pages=None):
    """A cache of random codes, scales and ring rows everywhere."""
    ref = Cache(n, per, kv, d, table, n_pages)
    ref.kc = rng.integers(-127, 128, ref.kc.shape).astype(np.int8)
    ref.vc = rng.integers(-127, 128, ref.vc.shape).astype(np.int8)
    ref.scales = (rng.uniform(0.3, 2.0, ref.scales.shape) / 60).astype(np.float32)
    ref.ring = rng.standard_normal(ref.ring.shape).astype(np.float32)
    return ref


def _attend(torch, ref, cache, q, starts, counts, heads, scale):
    from gpu_util import dev, empty_f32, host
    n, rows = q.shape[:2]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    out = empty_f32(n, rows, heads, ref.d)
    need = qlin.attend_kv8_workspace_bytes(n, rows, heads, ref.kv, ref.d, ref.per)
    ws = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device="cuda")  # (NaN wherever it is read before it is written)
    qlin.attend_kv8(cache, dev(q), out, rows, heads, i32(starts), None if counts is None else i32(counts), scale, ws)
    torch.cuda.synchronize()
    assert (ws[need:] == 0xFF).all()
    return host(out)


def _check_attend(torch, ref, cache, q, starts, counts, heads, scale):
    got = _attend(torch, ref, cache, q, starts, counts, heads, scale)
    n, rows = q.shape[:2]
    for s in range(n):
        c = rows if counts is None else max(0, min(counts[s], rows))
        k, v, there = ref.values(s, starts[s] + c)
        want, big = attend(q[s, :c].astype(np.float64), k, v, there, starts[s], scale)
        assert np.array_equal(np.isnan(got[s, :c]), np.isnan(want))
        err = np.nanmax(np.abs(got[s, :c] - want), initial=0.0)
        assert err <= attend_tolerance(big, v), (s, err, attend_tolerance(big, v))
        assert np.isnan(got[s, c:]).all()  # left as they were
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv", [(1, 1), (7, 1), (4, 2), (34, 2), (3, 3)])
@pytest.mark.parametrize("d", HEAD_DIMS)
def test_attend_one_row(heads, kv, d):
    """Every length around the borders of blocks and of 16-position tiles, from one position on."""
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(d + heads)
    ref = _filled(rng, 1, 9, kv, d)
    cache = _device_cache(torch, ref, paged=False)
    q = (1.5 * rng.standard_normal((1, 1, heads, d))).astype(np.float32)
    for start in (0, 1, 14, 15, 16, 17, 30, 31, 32, 33, 47, 63, 64, 200, 254, 255, 270, 286, 287):
        banner(f"attend d={d} heads={heads}/{kv} start={start}")
        _check_attend(torch, ref, cache, q, [start], None, heads, d ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,heads,kv,d,start", [(5, 8, 2, 64, 60), (33, 4, 2, 128, 0), (70, 3, 1, 96, 21), (64, 6, 2, 64, 64),
                                                   (130, 2, 2, 128, 90), (40, 8, 1, 256, 7), (90, 28, 4, 128, 100), (75, 5, 5, 192, 160),
                                                   (250, 4, 1, 64, 3), (200, 16, 1, 128, 37), (129, 32, 4, 64, 0)])
def test_attend_rows(rows, heads, kv, d, start):
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(rows + d)
    ref = _filled(rng, 1, (start + rows + 63) // 32, kv, d)
    cache = _device_cache(torch, ref, paged=False)
    banner(f"attend rows={rows} heads={heads}/{kv} d={d} start={start}")
    q = (1.5 * rng.standard_normal((1, rows, heads, d))).astype(np.float32)
    _check_attend(torch, ref, cache, q, [start], None, heads, d ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 37])
def test_attend_padded_batch(rows):
    """Ragged sequences, pages in no order, pages that are not there, starts outside the cache, empty sequences."""
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(rows)
    n, per, kv, d, heads = 9, 7, 2, 64, 6
    table = rng.permutation(n * per + 9)[:n * per].reshape(n, per)
    table[1, 0] = -1            # an evicted block
    table[2, :] = -7            # nothing is seen
    table[3, 6] = 1 << 30       # (the open block of a full cache)
    table[4, 1:3] = n * per + 9  # one past the last page
    ref = _filled(rng, n, per, kv, d, table, n * per + 9)
    cache = _device_cache(torch, ref, paged=True)
    q = rng.standard_normal((n, rows, heads, d)).astype(np.float32)
    for starts, counts in (([150, 60, 70, 200, 120, 0, 5, 223, 31], None),
                           ([100, 60, 0, 197, 90, 0, 5, 190, 64], [rows, 1, rows, rows, 0, rows, -1, 99, rows]),
                           ([-1, -2, -rows, -2 ** 31, 2 ** 31 - 1, 224, 230, 0, 1], None)):
        banner(f"attend padded rows={rows} starts={starts}")
        # a start past the capacity sees all of it
        got = _attend(torch, ref, cache, q, starts, counts, heads, 0.2)
        for s in range(n):
            c = rows if counts is None else max(0, min(counts[s], rows))
            start = min(starts[s], per * BLOCK)
            k, v, there = ref.values(s, start + c)
            want, big = attend(q[s, :c].astype(np.float64), k, v, there, start, 0.2)
            assert np.abs(got[s, :c] - want).max(initial=0.0) <= attend_tolerance(big, v), s
            assert np.isnan(got[s, c:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,heads,kv,d,length", [(1, 7, 1, 64, 9000), (2, 16, 2, 128, 5003), (1, 40, 1, 256, 3100), (20, 8, 1, 128, 2600)])
def test_attend_in_splits(rows, heads, kv, d, length):
    """Long caches, whose positions are split over workgroups and joined; one score far above the others in a split, a
    whole split far below."""
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(length)
    per = length // BLOCK + 2
    ref = _filled(rng, 1, per, kv, d)
    ref.scales[5:per // 2, :, 0] *= 1e-3
    ref.scales[per // 3, :, 0] *= 6
    ref.scales[per // 2:, :, 1] *= 1e-4
    cache = _device_cache(torch, ref, paged=False)
    assert qlin.attend_kv8_workspace_bytes(1, rows, heads, kv, d, per) > 0
    banner(f"attend length={length} heads={heads}/{kv} d={d}")
    q = rng.standard_normal((1, rows, heads, d)).astype(np.float32)
    _check_attend(torch, ref, cache, q, [length - rows], None, heads, d ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("n,rows,heads,kv,d,per", [
    (52, 1, 8, 4, 64, 9), (51, 2, 8, 4, 192, 5), (6, 70, 8, 2, 256, 6), (20, 37, 6, 2, 64, 7), (5, 70, 12, 4, 128, 9),
    (40, 31, 4, 4, 96, 5), (70, 1, 12, 4, 64, 30), (80, 19, 4, 4, 128, 5), (24, 1, 8, 4, 128, 40), (13, 3, 24, 4, 64, 60),
    (12, 5, 16, 2, 96, 50), (20, 1, 4, 4, 192, 70), (9, 2, 8, 4, 256, 70), (40, 1, 7, 1, 64, 140)])
def test_attend_many_sequences(n, rows, heads, kv, d, per):
    """Few and many rows of few and many sequences, from one block to all of them: each number of waves, splits and the
    joins of few and of many."""
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(n * rows + d)
    table = rng.permutation(n * per + 3)[:n * per].reshape(n, per)
    table[rng.random(table.shape) < 0.05] = -1
    ref = _filled(rng, n, per, kv, d, table, n * per + 3)
    cache = _device_cache(torch, ref, paged=True)
    starts = [int(x) for x in rng.integers(0, per * BLOCK - rows + 1, n)]
    starts[0], starts[-1] = per * BLOCK - rows, 0
    counts = [int(x) for x in rng.integers(0, rows + 1, n)]
    counts[0] = rows
    banner(f"attend n={n} rows={rows} heads={heads}/{kv} d={d} per={per}")
    q = rng.standard_normal((n, rows, heads, d)).astype(np.float32)
    _check_attend(torch, ref, cache, q, starts, counts, heads, d ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("n,rows,heads,kv,d", [(1, 250, 32, 8, 64), (1, 420, 28, 4, 64), (1, 500, 32, 8, 64), (70, 1, 12, 4, 64),
                                               (66, 1, 4, 4, 192), (48, 6, 12, 4, 128), (1, 110, 8, 2, 256), (80, 7, 12, 4, 96)])
def test_attend_long_caches(n, rows, heads, kv, d):
    """More than 64 blocks, with as many workgroups as CUs, more and fewer: split and not."""
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(n * rows + d)
    per = 72
    ref = _filled(rng, n, per, kv, d, rng.permutation(n * per).reshape(n, per), n * per)
    cache = _device_cache(torch, ref, paged=True)
    starts = [per * BLOCK - rows - 5] + [int(x) for x in rng.integers(0, per * BLOCK - rows, n - 1)]
    banner(f"attend n={n} rows={rows} heads={heads}/{kv} d={d} start={starts[0]}")
    q = rng.standard_normal((n, rows, heads, d)).astype(np.float32)
    _check_attend(torch, ref, cache, q, starts, None, heads, d ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40, 100])
def test_attend_odd_values(rows):
    """What a row does not see does not reach it, NaN and infinities among it; what it sees does."""
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(rows)
    kv, d, heads, per = 1, 64, 2, 6
    start = 64
    for where, place in (("a complete block", 2), ("a complete block", 3), ("the open block", None)):
        ref = _filled(rng, 1, per, kv, d)
        length = start + rows
        if place is not None:
            ref.scales[place, 0, 0] = np.nan
            ref.scales[place, 0, 1] = np.nan
        else:
            for p in range(length // BLOCK * BLOCK, length):
                if p >= length - 3:
                    ref.ring[0, 0, 0, p % RING, 1] = np.nan
                    ref.ring[0, 0, 1, p % RING, 2] = np.inf
            for p in range(length, per * BLOCK):  # rows that hold nothing yet
                ref.ring[0, 0, :, p % RING] = np.where(p >= length - length % BLOCK + BLOCK, ref.ring[0, 0, :, p % RING], np.nan)
        cache = _device_cache(torch, ref, paged=False)
        q = rng.standard_normal((1, rows, heads, d)).astype(np.float32)
        banner(f"attend odd values in {where} {place}, rows={rows}")
        with np.errstate(invalid="ignore"):
            got = _attend(torch, ref, cache, q, [start], None, heads, 0.3)
            k, v, there = ref.values(0, length)
            for r in range(rows):
                want, big = attend(q[0, r:r + 1].astype(np.float64), k, v, there, start + r, 0.3)
                dims = np.isfinite(want[0])
                assert np.array_equal(np.isfinite(got[0, r]), dims), (where, r)
                seen = v[:start + r + 1]
                assert np.abs(got[0, r] - want[0])[dims].max(initial=0.0) <= attend_tolerance(big, seen[np.isfinite(seen)]), (where, r)


@pytest.mark.gpu
def test_attend_large_and_small_scores():
    """Scores in the thousands (one position takes all) and of 1e-20 (all alike), and a head that is not a number alone."""
    torch = _gpu()
    from gpu_util import banner
    rng = np.random.default_rng(8)
    heads, kv, d = 4, 2, 128
    ref = _filled(rng, 1, 12, kv, d)
    cache = _device_cache(torch, ref, paged=False)
    for factor in (300.0, 1e-20, 1e-38):
        banner(f"scores times {factor}")
        q = (factor * rng.standard_normal((1, 2, heads, d))).astype(np.float32)
        _check_attend(torch, ref, cache, q, [370], None, heads, 0.5)
    q = rng.standard_normal((1, 2, heads, d)).astype(np.float32)
    q[0, 1, 2, 7] = np.inf
    banner("a query head with an infinity")
    got = _attend(torch, ref, cache, q, [370], None, heads, 0.5)
    k, v, there = ref.values(0, 372)
    want, big = attend(q[0, :1].astype(np.float64), k, v, there, 370, 0.5)
    assert np.isnan(got[0, 1, 2]).all()
    assert np.abs(got[0, 0] - want[0]).max() <= attend_tolerance(big, v)
    assert np.isfinite(got[0, 1, [0, 1, 3]]).all()


@pytest.mark.gpu
def test_attend_offsets_beyond_32_bits():
    """A page whose byte offset does not fit in 32 bits (4.5 GB of pages), in a table of two blocks."""
    torch = _gpu()
    from gpu_util import banner, dev
    rng = np.random.default_rng(1)
    kv, d, heads = 8, 256, 8
    rec = qlin.kv8_record_bytes(d)
    n_pages = (9 << 29) // (kv * rec)
    ref = _filled(rng, 1, 2, kv, d, np.array([[1, 0]]), 2)
    pages = torch.zeros(n_pages, kv, rec, dtype=torch.uint8, device="cuda")
    pages[n_pages - 2:] = dev(pack(ref.kc, ref.vc, ref.scales))
    table = torch.tensor([[n_pages - 1, n_pages - 2]], dtype=torch.int32, device="cuda")
    cache = qlin.Kv8Cache(pages, dev(ref.ring), table)
    banner("offsets beyond 32 bits")
    q = rng.standard_normal((1, 1, heads, d)).astype(np.float32)
    _check_attend(torch, ref, cache, q, [63], None, heads, d ** -0.5)
