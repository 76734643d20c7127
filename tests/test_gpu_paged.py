"""GPU tests of the paged cache: append with rotation, decode and prompt attention, against plain implementations in
64 bits on the values the device holds.

Tolerances. Rounding to bf16 is off by at most 2^-8 of the value (finfo(bf16).eps / 2).
* rotation: the 32-bit result differs from the exact one by a few 2^-24 of |x| + |y| and is rounded once, so an element is
  off by at most 2^-8 of itself plus 4 * 2^-24 * (|x| + |y|).
* attention: probabilities are rounded to 16 bits (2^-8 of each in bf16) before the product with V, whose sums and
  denominators are f32, and the result once more. With p_j the exact probabilities that is at most
  2^-8 * A + 2^-8 |o| per element, A = sum_j p_j |v_j|; the f32 terms (2^-22 relative in the exponentials, scores of up
  to 128 products with unit roundoff 2^-24 of sum |q||k|, tanh to 2^-22 of the cap) stay below a tenth of that for the
  scores of these tests (up to about 60), so 1.1 * (2^-8 * A + 2^-8 |o|) bounds every element.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pg():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    from maryml_b200 import paged
    return paged


# ---- plain forms ---------------------------------------------------------------------------
_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def fp4_values(codes, scales):
    table = torch.tensor(_E2M1 + [-x for x in _E2M1], dtype=torch.float64, device=codes.device)
    pair = torch.stack((codes & 15, codes >> 4), dim=-1).int()
    v = table[pair].reshape(*codes.shape[:-1], codes.shape[-1] // 8, 16)
    return (v * scales.view(torch.float8_e4m3fn).double().unsqueeze(-1)).flatten(-2)


class Setup:
    """A pool with every sequence's rows scattered over it; whatever no sequence owns is poison."""

    def __init__(self, pg, lens, page, kv_heads, d, nvfp4=False, seed=0, spare=3, poison=True, width=None):
        g = torch.Generator(device="cuda").manual_seed(1000 + seed)
        self.lens_host = list(lens)
        self.page, self.kvh, self.d, self.nvfp4 = page, kv_heads, d, nvfp4
        need = [-(-n // page) for n in lens]
        pages = sum(need) + spare
        perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        width = width or max(max(need), 1) + 2
        table = np.full((len(lens), width), -7, dtype=np.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = perm[at:at + n]
            at += n
        self.table = torch.from_numpy(table).cuda()
        self.lens = torch.tensor(self.lens_host, dtype=torch.int32, device="cuda")
        if nvfp4:
            mk = lambda: torch.randint(0, 256, (pages, page, kv_heads * d // 2), dtype=torch.uint8, device="cuda", generator=g)
            ms = lambda: torch.randint(0x28, 0x34, (pages, page, kv_heads * d // 16), dtype=torch.uint8, device="cuda", generator=g)
            planes = [mk(), mk(), ms(), ms()]
        else:
            mk = lambda: torch.randn((pages, page, kv_heads, d), device="cuda", generator=g).to(torch.bfloat16)
            planes = [mk(), mk()]
        if poison:
            keep = torch.zeros(pages * page, dtype=torch.bool)
            for b, n in enumerate(self.lens_host):
                r = torch.arange(n)
                keep[torch.from_numpy(table[b].astype(np.int64))[r // page] * page + r % page] = True
            gone = (~keep).cuda().view(pages, page)
            for t in planes[:2] if not nvfp4 else planes[2:]:
                t[gone] = float("nan") if not nvfp4 else 0x7F          # NaN rows; NaN scales
        self.cache = pg.PagedCache(planes[0], planes[1], *(planes[2:] or (None, None)), head_dim=d)
        self.gen = g

    def rows(self, b, name):
        """[len, kv_heads, d] in 64 bits."""
        n = self.lens_host[b]
        r = torch.arange(n, device="cuda")
        at = self.table[b].long()[r // self.page] * self.page + r % self.page
        if not self.nvfp4:
            return getattr(self.cache, name).reshape(-1, self.kvh, self.d)[at].double()
        codes = getattr(self.cache, name).reshape(-1, self.kvh * self.d // 2)[at]
        scales = getattr(self.cache, name + "_scales").reshape(-1, self.kvh * self.d // 16)[at]
        return fp4_values(codes, scales).view(n, self.kvh, self.d)


def plain_attention(q, k, v, pos, scale, softcap=0.0, window=0, slopes=None, prefix=0):
    """q [n, heads, d] at positions pos [n]; k, v [len, kv_heads, d], all 64 bits -> (o, A) with A = sum p |v|."""
    n, heads, d = q.shape
    length, kvh, _ = k.shape
    group = heads // kvh
    o, a = torch.zeros_like(q), torch.zeros_like(q)
    if length == 0:
        return o, a
    kpos = torch.arange(length, device=q.device)
    away = pos[:, None] - kpos[None]
    seen = away >= 0
    if window:
        seen &= away < window
    seen |= (kpos < prefix)[None]
    seen &= (pos >= 0)[:, None]
    for h in range(heads):
        x = q[:, h] @ k[:, h // group].t() * scale
        if softcap:
            x = softcap * torch.tanh(x / softcap)
        if slopes is not None:
            x = x - slopes[h].double() * away.abs()
        x = torch.where(seen, x, torch.full_like(x, -math.inf))
        p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
        o[:, h], a[:, h] = p @ v[:, h // group], p @ v[:, h // group].abs()
    return o, a


def check_attention(got, want, a):
    assert torch.isfinite(got.float()).all()
    err, room = (got.double() - want).abs(), 1.1 * 2.0 ** -8 * (a + want.abs()) + 1e-30
    worst = (err / room).max().item() if err.numel() else 0.0
    assert worst <= 1.0, worst
    return worst


def terms_of(s, heads, batch, softcap=0.0, window=0, slopes=False, prefix=None):
    kw = {"softcap": softcap, "window": window}
    if slopes:
        kw["slopes"] = torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda", dtype=torch.float32) / heads)
    if prefix is not None:
        kw["prefix"] = torch.tensor([prefix + 3 * b for b in range(batch)], dtype=torch.int32, device="cuda")
    return kw


def plain_terms(kw, b):
    return {"softcap": kw["softcap"], "window": kw["window"], "slopes": kw.get("slopes"),
            "prefix": int(kw["prefix"][b]) if "prefix" in kw else 0}


def run_decode(pg, s, heads, nq, gain=1.0, **t):
    batch = len(s.lens_host)
    q = (torch.randn((batch, nq, heads, s.d), device="cuda", generator=s.gen) * gain).to(torch.bfloat16)
    kw = terms_of(s, heads, batch, **t)
    got = pg.paged_attention_decode(q, s.cache, s.table, s.lens, **kw)
    torch.cuda.synchronize()
    worst = 0.0
    for b, n in enumerate(s.lens_host):
        pos = torch.arange(n - nq, n, device="cuda")
        o, a = plain_attention(q[b].double(), s.rows(b, "k"), s.rows(b, "v"), pos, 1.0 / math.sqrt(s.d), **plain_terms(kw, b))
        worst = max(worst, check_attention(got[b], o, a))
    return got, worst


def no_flags(pg):
    rc, flags = pg.context(0).check_flags()
    assert rc == 0, flags


# ---- decode ----------------------------------------------------------------------------------
@pytest.mark.parametrize("nvfp4", [False, True])
@pytest.mark.parametrize("lens,page,heads,kvh,d,nq", [
    ([1], 16, 8, 8, 128, 1),                            # one row, one query head per KV head
    ([64, 0, 1, 63, 65], 16, 8, 2, 128, 1),             # around a tile, and an empty sequence
    ([200, 777, 4, 1025], 48, 32, 8, 128, 1),           # pages that end inside tiles, several pieces
    ([5000], 64, 4, 1, 128, 1),                         # one KV head: the row is cut over many CTAs
    ([130, 2047, 300], 256, 16, 2, 64, 1),              # head_dim 64, all eight columns live
    ([33, 500], 80, 10, 1, 64, 1),                      # ten query heads over one KV head: two N tiles
    ([40, 900], 32, 48, 2, 128, 1),                     # twenty-four: two row tiles
    ([7, 128, 2, 600], 128, 8, 2, 128, 3),              # three tokens; a sequence shorter than that
    ([300, 9], 16, 5, 5, 64, 5),
])
def test_decode(pg, lens, page, heads, kvh, d, nq, nvfp4):
    run_decode(pg, Setup(pg, lens, page, kvh, d, nvfp4, seed=len(lens) + page), heads, nq)
    no_flags(pg)


@pytest.mark.parametrize("nvfp4", [False, True])
@pytest.mark.parametrize("terms", [
    {"softcap": 20.0}, {"window": 1}, {"window": 100}, {"window": 64, "prefix": 5}, {"slopes": True},
    {"softcap": 30.0, "window": 333, "prefix": 130, "slopes": True}, {"prefix": 10000}, {"window": 1 << 40},
])
def test_decode_terms(pg, terms, nvfp4):
    for d, heads, kvh, nq in ((128, 8, 2, 1), (64, 6, 1, 2), (128, 32, 2, 1)):
        run_decode(pg, Setup(pg, [700, 64, 129, 1, 0], 32, kvh, d, nvfp4, seed=nq), heads, nq, gain=4.0, **terms)
    no_flags(pg)


@pytest.mark.parametrize("terms", [{}, {"softcap": 30.0, "window": 333, "prefix": 130, "slopes": True}])
@pytest.mark.parametrize("kvh,d,group,nq", [(4, 128, 4, 1), (8, 64, 2, 2), (2, 128, 8, 1), (6, 64, 3, 1), (4, 128, 12, 1)])
def test_decode_nvfp4_heads_that_share_a_cta(pg, kvh, d, group, nq, terms):
    """A pool larger than half of L2: four KV heads (two where four does not divide) of a CTA read the same rows."""
    rows = int(62e6 / (kvh * d * 1.125))
    s = Setup(pg, [3000, 64, 0, 129, 1, 777], 256, kvh, d, nvfp4=True, seed=kvh, spare=rows // 256 + 1, width=rows // 256 + 20)
    run_decode(pg, s, kvh * group, nq, gain=3.0, **terms)
    no_flags(pg)


def test_decode_of_many_sequences_and_one_long_one(pg):
    """Lengths that differ by four orders of magnitude share the line of tiles; more than 32 sequences need the second
    round of the search for a CTA's first tile."""
    lens = [(37 * i) % 150 for i in range(100)] + [20000] + [1] * 30
    run_decode(pg, Setup(pg, lens, 64, 2, 128, seed=5), 8, 1)
    no_flags(pg)


def test_decode_evicted_pages_below_the_window_are_not_touched(pg):
    for nvfp4 in (False, True):
        s = Setup(pg, [1000, 555], 16, 2, 128, nvfp4, seed=3)
        q = torch.randn((2, 1, 8, 128), device="cuda", generator=s.gen).to(torch.bfloat16)
        want = pg.paged_attention_decode(q, s.cache, s.table, s.lens, window=100)
        cut = s.table.clone()
        cut[0, :(1000 - 100) // 16] = -1
        cut[1, :(555 - 100) // 16] = 1 << 30
        got = pg.paged_attention_decode(q, s.cache, cut, s.lens, window=100)
        assert torch.equal(got, want)
    no_flags(pg)


def test_decode_repeats_its_bits(pg):
    s = Setup(pg, [4097, 60, 1900, 4097], 16, 2, 128, seed=11)
    q = torch.randn((4, 1, 8, 128), device="cuda", generator=s.gen).to(torch.bfloat16)
    ref = pg.paged_attention_decode(q, s.cache, s.table, s.lens).clone()
    for _ in range(200):
        assert torch.equal(pg.paged_attention_decode(q, s.cache, s.table, s.lens), ref)


# ---- prompt ------------------------------------------------------------------------------------
def run_prompt(pg, s, heads, q_len, gain=1.0, pad=0, **t):
    batch, total = len(q_len), sum(q_len) + pad
    q = (torch.randn((total, heads, s.d), device="cuda", generator=s.gen) * gain).to(torch.bfloat16)
    cu = torch.tensor([0] + list(np.cumsum(q_len)), dtype=torch.int32, device="cuda")
    kw = terms_of(s, heads, batch, **t)
    out = torch.full_like(q, 7.0)
    got = pg.paged_attention_prompt(q, cu, s.cache, s.table, s.lens, out=out, **kw)
    torch.cuda.synchronize()
    assert got is out and (got[sum(q_len):] == 7.0).all()
    worst, t0 = 0.0, 0
    for b, n in enumerate(q_len):
        pos = torch.arange(s.lens_host[b] - n, s.lens_host[b], device="cuda")
        o, a = plain_attention(q[t0:t0 + n].double(), s.rows(b, "k"), s.rows(b, "v"), pos, 1.0 / math.sqrt(s.d), **plain_terms(kw, b))
        worst = max(worst, check_attention(got[t0:t0 + n], o, a))
        t0 += n
    return got, worst


PROMPTS = [
    # lens, q_len, page, heads, kvh, d
    ([1], [1], 16, 4, 1, 128),
    ([128], [128], 128, 1, 1, 128),                               # one tile, one head
    ([300, 5, 64], [300, 5, 64], 16, 8, 2, 128),                  # fresh ragged prompts, pages of 16
    ([1000, 0, 777, 130], [200, 0, 1, 130], 48, 32, 8, 128),      # chunks over a past, an empty one
    ([260, 700], [260, 99], 256, 10, 2, 128),                     # five heads per KV head: 125 of 128 rows in use
    ([513, 64], [513, 10], 32, 16, 4, 64),
    ([2000], [7], 64, 4, 4, 64),                                  # few blocks over many rows: the keys are cut
    ([3000, 40], [33, 20], 80, 4, 1, 128),
    ([90], [90], 16, 128, 1, 64),                                 # one token per tile
]


@pytest.mark.parametrize("nvfp4", [False, True])
@pytest.mark.parametrize("lens,q_len,page,heads,kvh,d", PROMPTS)
def test_prompt(pg, lens, q_len, page, heads, kvh, d, nvfp4):
    run_prompt(pg, Setup(pg, lens, page, kvh, d, nvfp4, seed=page + d), heads, q_len, pad=2)
    no_flags(pg)


@pytest.mark.parametrize("nvfp4", [False, True])
@pytest.mark.parametrize("terms", [
    {"softcap": 20.0}, {"window": 1}, {"window": 100}, {"window": 200, "prefix": 5}, {"slopes": True},
    {"softcap": 30.0, "window": 333, "prefix": 130, "slopes": True}, {"prefix": 10000}, {"prefix": 300, "slopes": True},
    {"window": 1 << 40},
])
def test_prompt_terms(pg, terms, nvfp4):
    for d, heads, kvh in ((128, 8, 2), (64, 6, 1)):
        run_prompt(pg, Setup(pg, [900, 64, 400, 1, 0], 32, kvh, d, nvfp4, seed=d), heads, [300, 64, 129, 1, 0], gain=4.0, **terms)
    run_prompt(pg, Setup(pg, [2500], 16, 1, 128, nvfp4, seed=8), 4, [40], gain=4.0, **terms)       # keys cut over CTAs
    no_flags(pg)


@pytest.mark.parametrize("gain,softcap", [(1.0, 50.0), (4.0, 50.0), (4.0, 12.0), (16.0, 20.0), (4.0, 1e-6), (4.0, 1e-3),
                                          (4.0, 355.0), (64.0, 355.0), (4.0, 1e4), (4.0, 1e8), (4.0, 1e18)])
def test_caps_of_every_size(pg, gain, softcap):
    """Scores far below the cap (where only the relative error of the tanh helps), near it and far beyond."""
    for d, heads in ((128, 4), (64, 2)):
        run_prompt(pg, Setup(pg, [700], 64, 1, d, seed=d + 1), heads, [300], gain=gain, softcap=softcap)
        run_decode(pg, Setup(pg, [700, 3], 64, 1, d, seed=d + 1), heads, 1, gain=gain, softcap=softcap)
    no_flags(pg)


def test_scales_and_caps_that_leave_f32_are_refused(pg):
    from maryml_b200 import MaryError
    s = Setup(pg, [20, 30], 16, 2, 128, seed=71)
    q, cu = torch.zeros((2, 1, 8, 128), dtype=torch.bfloat16, device="cuda"), torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for terms in ({"softcap": 3e38}, {"softcap": 1e19}, {"scale": 3e38}, {"scale": 1e19}):
        with pytest.raises(MaryError):
            pg.paged_attention_decode(q, s.cache, s.table, s.lens, **terms)
        with pytest.raises(MaryError):
            pg.paged_attention_prompt(q[:, 0], cu, s.cache, s.table, s.lens, **terms)
    no_flags(pg)


def test_prompt_scores_that_outgrow_their_reference(pg):
    """Keys whose scores rise by more than 2^40 towards the sequence's start, the last tiles to be read: every tile moves
    the running reference and rescales the output. The queries and keys are such that scores are exact."""
    for d in (64, 128):
        s = Setup(pg, [1500], 64, 1, d, seed=1, poison=False)
        k = s.cache.k.view(-1, d)
        rows = torch.arange(1500, device="cuda")
        at = s.table[0].long()[rows // 64] * 64 + rows % 64
        k[at] = 0
        step = (1500 - rows).float() // 32
        k[at, 0] = step.to(torch.bfloat16)                        # at most 46: exact
        q = torch.zeros((700, 2, d), device="cuda", dtype=torch.bfloat16)
        q[:, 0, 0], q[:, 1, 0] = 16.0, -16.0
        cu = torch.tensor([0, 700], dtype=torch.int32, device="cuda")
        got = pg.paged_attention_prompt(q, cu, s.cache, s.table, s.lens, scale=1.0)
        o, a = plain_attention(q.double(), s.rows(0, "k"), s.rows(0, "v"), torch.arange(800, 1500, device="cuda"), 1.0)
        check_attention(got, o, a)
    no_flags(pg)


def test_prompt_matches_decode_token_by_token(pg):
    s = Setup(pg, [300, 45], 16, 2, 128, seed=6)
    q = torch.randn((2, 1, 8, 128), device="cuda", generator=s.gen).to(torch.bfloat16)
    a = pg.paged_attention_decode(q, s.cache, s.table, s.lens)
    b = pg.paged_attention_prompt(q.view(2, 8, 128), torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), s.cache, s.table, s.lens)
    assert (a.view(2, 8, 128).float() - b.float()).abs().max() <= 2.0 ** -6 * a.float().abs().max()


# ---- append ----------------------------------------------------------------------------------
def plain_rotate(x, pos, inv_freq, sections=None):
    """x [n, heads, d] 64 bits; pos [axes, n] -> (rotated, |x| + |y| per element)."""
    d = x.shape[-1]
    f = inv_freq.double()
    if sections is None:
        angle = pos[0].double()[:, None] * f
    else:
        axis = np.repeat(np.arange(len(sections)), sections)
        angle = torch.stack([pos[int(a)].double() * f[i] for i, a in enumerate(axis)], dim=1)
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    lo, hi = x[..., :d // 2], x[..., d // 2:]
    size = (lo.abs() + hi.abs()).repeat(1, 1, 2)
    return torch.cat((lo * c - hi * s, hi * c + lo * s), -1), size


def inv_freq_of(d, theta=1e6):
    f = np.arange(d // 2, dtype=np.float64)
    return torch.from_numpy((1.0 / theta ** (2.0 * f / d)).astype(np.float32)).cuda()


def run_append(pg, s, hq, q_len, axes=0, ragged=True, far=0, pad=0, stride=0):
    """Appends q_len[b] tokens as the last rows of each sequence and checks queries, rows and untouched bytes."""
    d, kvh = s.d, s.kvh
    total = sum(q_len) + pad
    heads = hq + 2 * kvh
    wide = torch.randn((total, heads * d + stride), device="cuda", generator=s.gen).to(torch.bfloat16)
    qkv = wide[:, :heads * d]
    f = inv_freq_of(d)
    cu = torch.tensor([0] + list(np.cumsum(q_len)), dtype=torch.int32, device="cuda") if ragged else None
    kw = {}
    sections = None
    if axes:
        kw["positions"] = torch.randint(-50, 100000 + far, (axes, total), dtype=torch.int32, device="cuda", generator=s.gen)
        if axes > 1:
            left = d // 2
            sections = [left // axes + (1 if a < left % axes else 0) for a in range(axes)]
            kw["sections"] = tuple(sections)
    planes = {n: getattr(s.cache, n) for n in ("k", "v", "k_scales", "v_scales") if getattr(s.cache, n) is not None}
    before = {n: t.clone() for n, t in planes.items()}
    out = torch.full((total, hq, d), 7.0, dtype=torch.bfloat16, device="cuda")
    got = pg.paged_append(qkv, s.cache, s.table, s.lens, f, cu_q=cu, out=out, **kw)
    torch.cuda.synchronize()
    assert got.data_ptr() == out.data_ptr()
    x = qkv.double().reshape(total, heads, d)
    t0 = 0
    touched = torch.zeros(s.cache.pages * s.page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(q_len):
        row = torch.arange(s.lens_host[b] - n, s.lens_host[b], device="cuda")
        pos = kw["positions"][:, t0:t0 + n] if axes else row[None]
        rot, size = plain_rotate(x[t0:t0 + n, :hq + kvh], pos, f, sections)
        room = 2.0 ** -8 * rot.abs() + 4 * 2.0 ** -24 * size + 1e-30
        assert ((got[t0:t0 + n].double() - rot[:, :hq]).abs() <= room[:, :hq]).all()
        at = s.table[b].long()[row // s.page] * s.page + row % s.page
        touched[at] = True
        if not s.nvfp4:
            k = s.cache.k.reshape(-1, kvh, d)[at].double()
            assert ((k - rot[:, hq:]).abs() <= room[:, hq:]).all()
            assert torch.equal(s.cache.v.reshape(-1, kvh, d)[at], qkv.reshape(total, heads, d)[t0:t0 + n, hq + kvh:])
        t0 += n
    assert (got[t0:] == 7.0).all()
    for n, t in planes.items():
        same = (t.reshape(len(touched), -1).view(torch.uint8) == before[n].reshape(len(touched), -1).view(torch.uint8)).all(1)
        assert same[~touched].all(), n
    return qkv, got, touched, kw, cu


@pytest.mark.parametrize("lens,q_len,page,hq,kvh,d", [
    ([1], [1], 16, 4, 1, 128),
    ([300, 17, 5], [1, 1, 1], 16, 8, 2, 128),
    ([300, 17, 5, 64], [40, 0, 5, 64], 48, 5, 5, 64),
    ([2000, 900], [1500, 333], 128, 32, 8, 128),
    ([700, 0, 650], [700, 0, 650], 80, 7, 1, 64),
])
@pytest.mark.parametrize("axes", [0, 1, 3, 4])
def test_append(pg, lens, q_len, page, hq, kvh, d, axes):
    run_append(pg, Setup(pg, lens, page, kvh, d, seed=page), hq, q_len, axes, pad=3, stride=8 * axes)
    no_flags(pg)


def test_append_uniform_without_cu_q(pg):
    run_append(pg, Setup(pg, [5, 77, 130], 16, 2, 128, seed=2), 8, [4, 4, 4], ragged=False)
    no_flags(pg)


def test_append_far_positions(pg):
    """At a million rows the angle of the first frequency has lost six bits in f32; the kernel's has not."""
    run_append(pg, Setup(pg, [50], 16, 2, 128, seed=2), 4, [50], axes=1, far=2 ** 31 - 200000)


@pytest.mark.parametrize("d,kvh,page,q_len", [(128, 2, 32, [70, 1, 300]), (64, 3, 16, [1, 1, 1]), (128, 8, 64, [900, 300, 17])])
def test_append_nvfp4_rows_are_the_quantized_bf16_rows(pg, d, kvh, page, q_len):
    """Bit for bit: the bytes quantize_kv_rows gives for the rows a bf16 cache receives."""
    from maryml_b200.attention import quantize_kv_rows
    lens = [n + 11 * i for i, n in enumerate(q_len)]
    s4 = Setup(pg, lens, page, kvh, d, nvfp4=True, seed=4)
    qkv, got, touched, kw, cu = run_append(pg, s4, 4, q_len, axes=3)
    s16 = Setup(pg, lens, page, kvh, d, seed=4)
    assert torch.equal(s16.table, s4.table)
    q16 = pg.paged_append(qkv, s16.cache, s16.table, s16.lens, inv_freq_of(d), cu_q=cu, **kw)
    assert torch.equal(q16, got[:q16.shape[0]])
    for name in ("k", "v"):
        rows = getattr(s16.cache, name).reshape(-1, kvh, d)[touched].unsqueeze(0).contiguous()
        codes, scales = quantize_kv_rows(rows)
        assert torch.equal(getattr(s4.cache, name).reshape(-1, kvh * d // 2)[touched], codes[0])
        assert torch.equal(getattr(s4.cache, name + "_scales").reshape(-1, kvh * d // 16)[touched], scales[0])


# ---- bad tables and lengths -----------------------------------------------------------------------
@pytest.mark.parametrize("nvfp4", [False, True])
def test_bad_entries_are_contained_and_flagged(pg, nvfp4):
    s = Setup(pg, [100, 90, 80], 16, 2, 128, nvfp4, seed=9, poison=False)
    q = torch.randn((3, 1, 8, 128), device="cuda", generator=s.gen).to(torch.bfloat16)
    want = pg.paged_attention_decode(q, s.cache, s.table, s.lens).clone()
    no_flags(pg)
    bad = s.table.clone()
    bad[1, 2] = -5
    got = pg.paged_attention_decode(q, s.cache, bad, s.lens)
    rc, flags = pg.context(0).check_flags()
    assert rc != 0 and flags[2] == 2
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2]) and torch.isfinite(got.float()).all()
    # the page reads as zeros
    k, v = s.rows(1, "k"), s.rows(1, "v")
    k[32:48], v[32:48] = 0, 0
    o, a = plain_attention(q[1].double(), k, v, torch.tensor([89], device="cuda"), 1 / math.sqrt(128))
    check_attention(got[1], o, a)
    # lengths beyond the table are clamped to it (the entries it has there are no pages), negative ones to zero
    for value in (10 ** 9, -4):
        lens = s.lens.clone()
        lens[2] = value
        got = pg.paged_attention_decode(q, s.cache, s.table, lens)
        rc, flags = pg.context(0).check_flags()
        assert rc != 0 and flags[2] == 3, flags
        assert torch.equal(got[:2], want[:2]) and torch.isfinite(got.float()).all()
        assert value > 0 or (got[2] == 0).all()
    # an append has nowhere to go: nothing is written
    planes = [t for t in (s.cache.k, s.cache.v, s.cache.k_scales, s.cache.v_scales) if t is not None]
    before = [t.clone() for t in planes]
    qkv = torch.randn((3, 12 * 128), device="cuda", generator=s.gen).to(torch.bfloat16)
    bad = torch.full_like(s.table, s.cache.pages)
    pg.paged_append(qkv, s.cache, bad, s.lens, inv_freq_of(128))
    rc, flags = pg.context(0).check_flags()
    assert rc != 0 and flags[2] in (1, 2, 3)
    assert all(torch.equal(t, u) for t, u in zip(planes, before))


# ---- the operators together, as a server uses them ---------------------------------------------------
def test_serving_run_with_a_replayed_step(pg):
    """Ragged prompts in two chunks, then decode steps replayed from one captured graph while lengths and tables grow on the
    device; every attention output against the plain form on the rows the cache then holds."""
    hq, kvh, d, page, batch = 8, 2, 128, 16, 3
    chunks = [[37, 100, 5], [20, 61, 0]]
    steps = 20
    ends = [sum(c[b] for c in chunks) + steps for b in range(batch)]
    s = Setup(pg, ends, page, kvh, d, seed=21)
    full_table = s.table.clone()
    f = inv_freq_of(d)
    heads = hq + 2 * kvh
    done = [0] * batch
    for c in chunks:
        qkv = torch.randn((sum(c), heads * d), device="cuda", generator=s.gen).to(torch.bfloat16)
        cu = torch.tensor([0] + list(np.cumsum(c)), dtype=torch.int32, device="cuda")
        done = [a + n for a, n in zip(done, c)]
        lens = torch.tensor(done, dtype=torch.int32, device="cuda")
        q = pg.paged_append(qkv, s.cache, s.table, lens, f, cu_q=cu)
        out = pg.paged_attention_prompt(q, cu, s.cache, s.table, lens, window=70)
        s.lens_host = list(done)
        t0 = 0
        for b, n in enumerate(c):
            pos = torch.arange(done[b] - n, done[b], device="cuda")
            o, a = plain_attention(q[t0:t0 + n].double(), s.rows(b, "k"), s.rows(b, "v"), pos, 1.0 / math.sqrt(d), window=70)
            check_attention(out[t0:t0 + n], o, a)
            t0 += n
    # a step on static buffers: lengths and table are rewritten between replays (pages appear as they are needed)
    lens = torch.tensor(done, dtype=torch.int32, device="cuda")
    table = torch.full_like(full_table, -1)
    qkv = torch.zeros((batch, heads * d), dtype=torch.bfloat16, device="cuda")
    stream = torch.cuda.Stream()

    def step():
        lens.add_(1)
        q = pg.paged_append(qkv, s.cache, table, lens, f)
        return q, pg.paged_attention_decode(q.view(batch, 1, hq, d), s.cache, table, lens, window=70)

    def fill(upto):
        for b, n in enumerate(upto):
            table[b, :-(-n // page)] = full_table[b, :-(-n // page)]

    fill([n + 1 for n in done])
    with torch.cuda.stream(stream):
        stream.wait_stream(torch.cuda.default_stream())
        step()                                             # warm-up: this row is written again by the first replay
        lens.sub_(1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        q, out = step()
    for i in range(steps):
        fill([n + 1 for n in done])
        qkv.copy_(torch.randn((batch, heads * d), device="cuda", generator=s.gen))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        done = [n + 1 for n in done]
        assert lens.tolist() == done
        s.lens_host = list(done)
        for b in range(batch):
            at = int(full_table[b, (done[b] - 1) // page]) * page + (done[b] - 1) % page
            assert torch.equal(s.cache.v.view(-1, kvh, d)[at], qkv.view(batch, heads, d)[b, hq + kvh:])
            o, a = plain_attention(q[b:b + 1].double(), s.rows(b, "k"), s.rows(b, "v"), torch.tensor([done[b] - 1], device="cuda"),
                                   1.0 / math.sqrt(d), window=70)
            check_attention(out[b], o, a)
    no_flags(pg)


def test_layer_over_a_paged_cache(pg):
    """forward_paged is its parts in order, bit for bit; and its first layer of arithmetic is forward's: the rows it appends
    are the contiguous cache's up to the rounding points of the rotation."""
    from maryml_b200 import layer, nvfp4 as nv
    cfg = layer.LayerConfig(hidden=512, heads=4, kv_heads=2, head_dim=128, inter=1024)
    g = torch.Generator(device="cuda").manual_seed(3)
    full = {}
    for name, n, k in (("q", 512, 512), ("k", 256, 512), ("v", 256, 512), ("o", 512, 512), ("gate", 1024, 512), ("up", 1024, 512),
                       ("down", 512, 1024)):
        w = (torch.randn((n, k), device="cuda", generator=g) * 0.02).to(torch.bfloat16)
        p = nv.Nvfp4.quantize(w)
        full[name] = (p.codes, p.scales, p.scale2)
    gain = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    L = layer.DecoderLayer(cfg, full, gain, gain)
    q_len = [70, 33]
    lens = [70, 50]
    s = Setup(pg, lens, 16, 2, 128, seed=31)
    x = torch.randn((sum(q_len), 512), device="cuda", generator=g).to(torch.bfloat16)
    cu = torch.tensor([0, 70, 103], dtype=torch.int32, device="cuda")
    y = L.forward_paged(x, s.cache, s.table, s.lens, cu_q=cu, softcap=30.0)
    _, xq = L._norm_quantize(x, None, L.input_gain)
    qkv = nv.gemm_w4a4_stacked(xq[0], xq[1], L.wqkv, xq[2])
    q = pg.paged_append(qkv, s.cache, s.table, s.lens, L.inv_freq, cu_q=cu)
    a = pg.paged_attention_prompt(q, cu, s.cache, s.table, s.lens, softcap=30.0)
    o_sum = L._linear(a.reshape(103, 512), L.wo, out_dtype=torch.float32)
    residual, down = L.half_mlp(x, o_sum, down_dtype=torch.bfloat16)
    assert torch.equal(y, layer.add(residual, down))
    # the contiguous layer's rows of the fresh sequence
    kc, vc = (torch.zeros((1, 70, 2, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    L.forward(x[:70], 1, 0, kc, vc)
    assert torch.equal(s.rows(0, "v"), vc[0].double())
    # forward rounds cos and sin to bf16 (2^-8 of each), both products and the sum: 2^-8 * 3 of |x| + |y|, and paged_append's one
    size = (kc[0].double()[..., :64].abs() + kc[0].double()[..., 64:].abs()).repeat(1, 1, 2) * math.sqrt(2.0)
    assert ((s.rows(0, "k") - kc[0].double()).abs() <= 4 * 2.0 ** -8 * size).all()
    # a decode step of one token each
    s.lens.add_(0)
    y1 = L.forward_paged(x[:2], s.cache, s.table, s.lens)
    q = pg.paged_append(nv.gemm_w4a4_stacked(*L._quantize(layer.rmsnorm(x[:2], L.input_gain, cfg.eps))[:2], L.wqkv, 2), s.cache,
                        s.table, s.lens, L.inv_freq)
    a = pg.paged_attention_decode(q.view(2, 1, 4, 128), s.cache, s.table, s.lens)
    residual, down = L.half_mlp(x[:2], L._linear(a.view(2, 512), L.wo, out_dtype=torch.float32), down_dtype=torch.bfloat16)
    assert torch.equal(y1, layer.add(residual, down))
    with pytest.raises(ValueError):
        layer.DecoderLayer(cfg, full, gain, gain, fuse=False).forward_paged(x, s.cache, s.table, s.lens, cu_q=cu)
    no_flags(pg)


def test_another_stream_and_overlapping_calls(pg):
    """Two streams at once, each with its own workspace from the allocator: both as alone."""
    setups = [Setup(pg, [3000 + 7 * i, 40, 900], 64, 2, 128, seed=40 + i) for i in range(2)]
    qs = [torch.randn((3, 1, 8, 128), device="cuda", generator=s.gen).to(torch.bfloat16) for s in setups]
    qp = [torch.randn((130, 8, 128), device="cuda", generator=s.gen).to(torch.bfloat16) for s in setups]
    cu = torch.tensor([0, 90, 130, 130], dtype=torch.int32, device="cuda")
    want = [(pg.paged_attention_decode(q, s.cache, s.table, s.lens), pg.paged_attention_prompt(p, cu, s.cache, s.table, s.lens))
            for s, q, p in zip(setups, qs, qp)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                s = setups[i]
                got[i].append((pg.paged_attention_decode(qs[i], s.cache, s.table, s.lens),
                               pg.paged_attention_prompt(qp[i], cu, s.cache, s.table, s.lens)))
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in got[i]:
            assert torch.equal(a, want[i][0]) and torch.equal(b, want[i][1])
    no_flags(pg)


def test_strided_tables_and_kept_workspace(pg):
    s = Setup(pg, [500, 77], 16, 2, 128, seed=50)
    wide = torch.full((2, s.table.shape[1] + 9), 1 << 29, dtype=torch.int32, device="cuda")
    wide[:, 4:4 + s.table.shape[1]] = s.table
    view = wide[:, 4:4 + s.table.shape[1]]
    q = torch.randn((2, 1, 8, 128), device="cuda", generator=s.gen).to(torch.bfloat16)
    want = pg.paged_attention_decode(q, s.cache, s.table, s.lens)
    ws = torch.full((64 << 20,), 0xFF, dtype=torch.uint8, device="cuda")          # its contents do not matter
    out = torch.empty_like(q)
    for _ in range(3):
        assert pg.paged_attention_decode(q, s.cache, view, s.lens, out=out, workspace=ws) is out
        assert torch.equal(out, want)
    no_flags(pg)


def test_an_sm_limit_changes_the_cut_not_the_result(pg):
    from maryml_b200 import _lib
    s = Setup(pg, [9000, 100], 64, 2, 128, seed=51)
    q = torch.randn((2, 1, 8, 128), device="cuda", generator=s.gen).to(torch.bfloat16)
    a = pg.paged_attention_decode(q, s.cache, s.table, s.lens)
    ctx = pg.context(0)
    ctx.check(_lib.lib.mb_ctx_set_sm_limit(ctx.handle, 20))
    try:
        b = pg.paged_attention_decode(q, s.cache, s.table, s.lens)
    finally:
        ctx.check(_lib.lib.mb_ctx_set_sm_limit(ctx.handle, 0))
    o, room = plain_attention(q[0].double(), s.rows(0, "k"), s.rows(0, "v"), torch.tensor([8999], device="cuda"), 1 / math.sqrt(128))
    check_attention(a[0], o, room)
    check_attention(b[0], o, room)


def test_a_pool_beyond_two_to_the_32_bytes(pg):
    """Rows past 2^31 elements and 2^32 bytes of a pool are addressed in 64 bits, by the append and by both readers."""
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB of free device memory")
    for nvfp4 in (False, True):
        kvh, d, page = 8, 128, 256
        pages = (5 << 30) // (page * kvh * d * 2) if not nvfp4 else (5 << 30) // (page * kvh * d // 2)
        cache = pg.PagedCache.empty(pages, page, kvh, d, nvfp4=nvfp4)
        n = 300
        table = torch.tensor([[pages - 1, pages - 3, -1], [1, pages // 2, -1]], dtype=torch.int32, device="cuda")
        lens = torch.tensor([n, n - 7], dtype=torch.int32, device="cuda")
        g = torch.Generator(device="cuda").manual_seed(5)
        hq = 8
        qkv = torch.randn((2 * n - 7, (hq + 2 * kvh) * d), device="cuda", generator=g).to(torch.bfloat16)
        cu = torch.tensor([0, n, 2 * n - 7], dtype=torch.int32, device="cuda")
        q = pg.paged_append(qkv, cache, table, lens, inv_freq_of(d), cu_q=cu)
        out = pg.paged_attention_prompt(q, cu, cache, table, lens)
        one = pg.paged_attention_decode(torch.stack((q[n - 1], q[-1])).unsqueeze(1), cache, table, lens)
        for b, (length, t0) in enumerate(((n, 0), (n - 7, n))):
            r = torch.arange(length, device="cuda")
            page_of, row = table[b].long()[r // page], r % page
            if nvfp4:
                k, v = (fp4_values(getattr(cache, x)[page_of, row], getattr(cache, x + "_scales")[page_of, row]).view(length, kvh, d)
                        for x in ("k", "v"))
            else:
                k, v = cache.k[page_of, row].double(), cache.v[page_of, row].double()
                assert torch.equal(cache.v[page_of, row], qkv.view(-1, hq + 2 * kvh, d)[t0:t0 + length, hq + kvh:])
            o, a = plain_attention(q[t0:t0 + length].double(), k, v, r, 1 / math.sqrt(d))
            check_attention(out[t0:t0 + length], o, a)
            check_attention(one[b], o[-1:], a[-1:])
        del cache
    no_flags(pg)


def test_masked_keys_may_hold_anything(pg):
    """NaN and infinities in rows nobody sees: behind the length, below a window, in pages of others. Keys a query does not
    see may be NaN or infinite too (their scores are replaced before they are used)."""
    for d in (64, 128):
        s = Setup(pg, [200, 130], 32, 2, d, seed=60)
        at = lambda b, r: int(s.table[b, r // 32]) * 32 + r % 32
        k, v = s.cache.k.view(-1, 2, d), s.cache.v.view(-1, 2, d)
        q = torch.randn((2, 1, 8, d), device="cuda", generator=s.gen).to(torch.bfloat16)
        want = pg.paged_attention_decode(q, s.cache, s.table, s.lens, window=50).clone()
        for r in range(0, 150):
            k[at(0, r)] = float("inf") if r % 2 else float("nan")
            v[at(0, r)] = float("nan") if r % 2 else float("-inf")
        assert torch.equal(pg.paged_attention_decode(q, s.cache, s.table, s.lens, window=50), want)
    no_flags(pg)


def test_nan_in_a_key_that_is_seen_comes_out(pg):
    """A NaN in a row of K makes the rows that see it NaN, alone or among others, in one piece or joined, and no other row."""
    for d in (64, 128):
        for softcap in (0.0, 20.0):
            s = Setup(pg, [40, 1, 2000, 7], 32, 2, d, seed=62)
            row = lambda b, r: int(s.table[b, r // 32]) * 32 + r % 32
            k = s.cache.k.view(-1, 2, d)
            for b, r in ((0, 17), (1, 0), (2, 1234)):
                k[row(b, r), 0, 3] = float("nan")                 # the first KV head only
            q = torch.randn((4, 1, 8, d), device="cuda", generator=s.gen).to(torch.bfloat16)
            cu = torch.arange(5, dtype=torch.int32, device="cuda")
            for out in (pg.paged_attention_decode(q, s.cache, s.table, s.lens, softcap=softcap).view(4, 8, d),
                        pg.paged_attention_prompt(q.view(4, 8, d), cu, s.cache, s.table, s.lens, softcap=softcap)):
                assert out[:3, :4].isnan().all() and out[3].isfinite().all() and out[:, 4:].isfinite().all()
    no_flags(pg)


def test_zero_tokens_are_a_call_that_does_nothing(pg):
    s = Setup(pg, [5, 6], 16, 2, 128, seed=61)
    cu = torch.zeros(3, dtype=torch.int32, device="cuda")
    q = pg.paged_append(torch.empty((0, 12 * 128), dtype=torch.bfloat16, device="cuda"), s.cache, s.table, s.lens, inv_freq_of(128), cu_q=cu)
    assert q.shape == (0, 8, 128)
    assert pg.paged_attention_prompt(q, cu, s.cache, s.table, s.lens).shape == (0, 8, 128)
    no_flags(pg)


def test_refusals(pg):
    from maryml_b200 import MaryError
    s = Setup(pg, [20, 30], 16, 2, 128, seed=70)
    q = torch.zeros((2, 1, 8, 128), dtype=torch.bfloat16, device="cuda")
    qp, cu = q.view(2, 8, 128), torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    qkv = torch.zeros((2, 12 * 128), dtype=torch.bfloat16, device="cuda")
    f = inv_freq_of(128)
    dec = lambda **k: pg.paged_attention_decode(k.pop("q", q), k.pop("cache", s.cache), k.pop("t", s.table), k.pop("n", s.lens), **k)
    pro = lambda **k: pg.paged_attention_prompt(k.pop("q", qp), k.pop("cu", cu), k.pop("cache", s.cache), k.pop("t", s.table), k.pop("n", s.lens), **k)
    app = lambda **k: pg.paged_append(k.pop("x", qkv), k.pop("cache", s.cache), k.pop("t", s.table), k.pop("n", s.lens), k.pop("f", f), **k)
    bad_page = pg.PagedCache(*(torch.zeros((4, 24, 2, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    bad_dim = pg.PagedCache(*(torch.zeros((4, 16, 2, 96), dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    cases = [
        lambda: dec(q=q.float()), lambda: dec(q=q[:, :, :, :64]), lambda: dec(q=q[:1]), lambda: dec(q=torch.zeros((2, 1, 7, 128), dtype=torch.bfloat16, device="cuda")),
        lambda: dec(t=s.table.long()), lambda: dec(t=s.table.t()), lambda: dec(t=s.table.cpu()), lambda: dec(n=s.lens[:1]), lambda: dec(n=s.lens.long()),
        lambda: dec(scale=-1.0), lambda: dec(scale=float("nan")), lambda: dec(scale=0.0), lambda: dec(softcap=-1.0), lambda: dec(softcap=float("inf")), lambda: dec(softcap=1e-40), lambda: dec(softcap=1e40), lambda: dec(window=1 << 70), lambda: dec(window=1.5),
        lambda: dec(window=-3), lambda: dec(slopes=torch.zeros(7, device="cuda")), lambda: dec(slopes=torch.zeros(8, dtype=torch.float64, device="cuda")),
        lambda: dec(prefix=torch.zeros(3, dtype=torch.int32, device="cuda")), lambda: dec(prefix=torch.zeros(2, device="cuda")),
        lambda: dec(out=torch.zeros((2, 8, 128), dtype=torch.bfloat16, device="cuda")), lambda: dec(cache=bad_page),
        lambda: dec(cache=bad_dim, q=torch.zeros((2, 1, 8, 96), dtype=torch.bfloat16, device="cuda")), lambda: dec(t=s.table[:, :0]),
        lambda: pro(q=qp.float()), lambda: pro(q=q), lambda: pro(cu=cu[:2]), lambda: pro(cu=cu.long()), lambda: pro(cu=cu.cpu()),
        lambda: pro(scale=0.0), lambda: pro(cache=bad_page), lambda: pro(q=torch.zeros((2, 258, 128), dtype=torch.bfloat16, device="cuda")),
        lambda: app(x=qkv.float()), lambda: app(x=qkv[:, :-1]), lambda: app(x=qkv[:, :4 * 128]), lambda: app(x=qkv.t()), lambda: app(f=f[:32]), lambda: app(f=f.double()),
        lambda: app(cu_q=cu[:2]), lambda: app(x=torch.zeros((3, 12 * 128), dtype=torch.bfloat16, device="cuda")), lambda: app(sections=(64,)),
        lambda: app(positions=torch.zeros((3, 2), dtype=torch.int32, device="cuda")), lambda: app(positions=torch.zeros((3, 2), dtype=torch.int32, device="cuda"), sections=(16, 24, 23)),
        lambda: app(positions=torch.zeros((5, 2), dtype=torch.int32, device="cuda"), sections=(16, 24, 24, 0, 0)), lambda: app(positions=torch.zeros((1, 3), dtype=torch.int32, device="cuda")),
        lambda: app(x=torch.zeros((2, 12 * 128 + 4), dtype=torch.bfloat16, device="cuda")[:, :12 * 128]), lambda: app(cache=bad_page),
        lambda: pg.PagedCache(s.cache.k, s.cache.v[:1]), lambda: pg.PagedCache(s.cache.k.float(), s.cache.v.float()),
        lambda: pg.PagedCache(s.cache.k.transpose(1, 2), s.cache.v.transpose(1, 2)), lambda: pg.PagedCache(s.cache.k, s.cache.v, head_dim=64),
        lambda: pg.PagedCache(s.cache.k.view(torch.uint8), s.cache.v.view(torch.uint8), s.cache.k, None, head_dim=128),
    ]
    for i, c in enumerate(cases):
        with pytest.raises(MaryError):
            c()
            pytest.fail(f"case {i} was not refused")
    no_flags(pg)
