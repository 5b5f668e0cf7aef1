"""The quantized K/V cache on the GPU against the formulas in 64 bits.

Tolerances.  Held values are compared exactly: codes and scales are fixed by
the format.  For the attention, with e_t = torch.finfo(t).eps / 2 the half
step of q's type, A = sum_j p_j |v_j| / sum_j p_j and K = scale * max_j sum_d
|q_d k_jd|, an output may be off by

    e_t max(|out|, tiny_t) + (P + 2 * 2^-18 K + 2^-18) A + 2^-39 n max |v|

* the first term is the rounding to q's type; below the smallest normal
  number tiny_t its steps stay those at tiny_t, 2 e_t tiny_t (fp16: 2^-24);
* P: for 16-bit types the probabilities enter the tensor cores as one fp16
  each, and so may the 8-bit values and keys: three roundings of 2^-11 at most
  on a product p_j v_j; for fp32 as fp16 pairs, 2^-20;
* 2^-18 K bounds the fp32 error of a score, up to 2^6 additions each off by
  2^-24 of the sum of magnitudes; an error of a score is a relative error of
  its p and of the sum of p, so it counts twice.  For 16-bit types the rounding
  of 8-bit keys to fp16 adds up to 2^-11 K, also twice;
* 2^-18: sums of p and p v in fp32, exp2 and the final division;
* a product p_j s_j, taken relative to the largest p and s so that it lies
  below 2^15, is never held finer than fp16's last half step 2^-25: 2^-40 of
  the largest, and s_j times a code is at most max |v|; n terms, doubled.
"""

import math

import pytest
import torch

from qwen_megakernel_b200 import KVCacheError, KVRows, QuantKVCache

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def held(x, bits):
    """The values that rows x stand for once held, in 64 bits."""
    top = 7 if bits == 4 else 127
    g = x.double().unflatten(-1, (-1, 32))
    fin = torch.where(g.isfinite(), g, 0.0)
    s = (fin.abs().amax(-1, keepdim=True) / top).bfloat16().double()
    c = (g / torch.where(s > 0, s, 1.0)).round().clamp(-top, top)
    c = torch.where((s > 0) & ~g.isnan(), c, 0.0)
    return (c * s).flatten(-2)


def attention(q, k, v, limits, scale):
    """Rows q [n, hq, d] over k, v [m, hk, d] (64 bits); row i sees limits[i]
    positions.  Returns out and sum_j p |v| / sum_j p."""
    n, hq, d = q.shape
    ratio = hq // k.shape[1]
    k, v = k.repeat_interleave(ratio, 1), v.repeat_interleave(ratio, 1)
    s = torch.einsum("nhd,mhd->hnm", q.double(), k) * scale
    live = torch.arange(k.shape[0], device=q.device)[None, :] < torch.as_tensor(limits, device=q.device)[:, None]
    p = torch.softmax(s.masked_fill(~live, -math.inf), -1)
    return torch.einsum("hnm,mhd->nhd", p, v), torch.einsum("hnm,mhd->nhd", p, v.abs())


def check_attend(got, q, k, v, limits, bits, scale):
    """got against the formulas."""
    ref, A = attention(q, k, v, limits, scale)
    seen = k[:max(limits)].abs().repeat_interleave(q.shape[1] // k.shape[1], 1)
    K = abs(scale) * torch.einsum("nhd,mhd->nhm", q.double().abs(), seen).amax(-1, keepdim=True)
    low = q.dtype != torch.float32
    P = 3 * 2.0**-11 if low else 2.0**-20
    if low and bits == 8:
        P = P + 2 * 2.0**-11 * K
    e = torch.finfo(q.dtype).eps / 2
    tol = e * ref.abs().clamp(min=torch.finfo(q.dtype).tiny) + (P + 2 * 2.0**-18 * K + 2.0**-18) * A + 2.0**-39 * max(limits) * v.abs().max()
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off; worst "
                           f"{((got.double() - ref).abs() / tol).max().item():.2f} of the tolerance")
    assert torch.isfinite(got).all()


class Filled:
    """A cache whose sequences hold random rows, and the rows."""

    def __init__(self, lens, hk=2, d=128, bits=4, dtype=torch.bfloat16, seed=0, max_seq_len=None, layers=1, layer=0,
                 v_gain=0.7):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.cache = QuantKVCache(len(lens), max_seq_len or max(lens), num_layers=layers, num_kv_heads=hk, head_dim=d,
                                  bits=bits)
        self.bits, self.layer, self.gen = bits, layer, g
        self.k, self.v = [], []
        for n in lens:
            self.k.append(torch.randn(n, hk, d, generator=g, device="cuda").mul_(1.3).to(dtype))
            self.v.append(torch.randn(n, hk, d, generator=g, device="cuda").mul_(v_gain).to(dtype))
        self.cache.write(torch.cat(self.k), torch.cat(self.v), KVRows([0] * len(lens), lens), layer)
        self.cache.check_status()

    def check(self, got, q, segs, scale=None):
        """segs: (seq, start, count) of got's and q's rows."""
        scale = scale or 1 / math.sqrt(q.shape[-1])
        r = 0
        for seq, start, n in segs:
            if n:
                k = held(self.k[seq], self.bits)
                v = held(self.v[seq], self.bits)
                check_attend(got[r:r + n], q[r:r + n], k, v, [start + i + 1 for i in range(n)], self.bits, scale)
            r += n


# ---------------------------------------------------------- write and read
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128])
def test_write_read_exact(dtype, bits, d):
    """Segments of 0, 1 and several rows; values at and next to rounding
    borders, groups of zeros, subnormals and the type's largest values."""
    g = torch.Generator(device="cuda").manual_seed(d + bits)
    counts, starts, seqs = [1, 0, 9, 70], [37, 5, 0, 130], [3, 2, 1, 0]
    n, hk = sum(counts), 3
    x = torch.randn(2, n, hk, d, generator=g, device="cuda", dtype=torch.float64)
    x *= torch.exp(3 * torch.randn(2, n, hk, d // 32, 1, generator=g, device="cuda", dtype=torch.float64)).expand(
        -1, -1, -1, -1, 32).flatten(-2)
    top = 7 if bits == 4 else 127
    ties = (torch.arange(d, device="cuda") % (top + 1)) + 0.5  # (c + 1/2) s with s = 1
    ties[::32] = top
    x[0, 10] = ties
    x[0, 11] = -ties * 2.0**-9
    x[1, 12] = 0.0
    x[1, 13, :, :32] = 0.0
    fi = torch.finfo(dtype)
    x[0, 14] = fi.max * torch.sign(x[0, 14])
    x[0, 15] = fi.tiny * x[0, 15].abs().clamp(max=1.0)
    x[0, 16] = fi.tiny * fi.eps * torch.randint(-200, 200, (hk, d), generator=g, device="cuda")
    k, v = x[0].to(dtype), x[1].to(dtype)
    if dtype == torch.float32:  # neighbours of borders
        k[17] = torch.nextafter(k[10], torch.full_like(k[10], 100.0))
        k[18] = torch.nextafter(k[10], torch.full_like(k[10], -100.0))
        k[17:19, :, ::32] = top
    cache = QuantKVCache(4, 200, num_layers=2, num_kv_heads=hk, head_dim=d, bits=bits)
    rows = KVRows(starts, counts, seqs)
    cache.write(k, v, rows, layer=1)
    for t in TYPES:
        kr, vr = cache.read(rows, layer=1, dtype=t)
        # exact values have at most 15 bits: one rounding, to t
        assert torch.equal(kr, held(k, bits).float().to(t)) and torch.equal(vr, held(v, bits).float().to(t))
    # (some of the spread values lie past fp16's range: infinities, reported)
    if torch.isfinite(k).all() and torch.isfinite(v).all():
        cache.check_status()
    else:
        with pytest.raises(KVCacheError, match="NaN or infinity"):
            cache.check_status()
    # nothing else was written: the other layer, and the other positions
    assert not cache.k_codes[:, 0].any() and not cache.v_scales[:, 0].any()
    live = torch.zeros(4, 256, dtype=torch.bool)
    for s, c, q in zip(starts, counts, seqs):
        live[q, s:s + c] = True
    assert not cache.k_codes[:, 1].transpose(1, 2)[~live.cuda()].any()
    assert not cache.v_codes[:, 1].transpose(1, 2)[~live.cuda()].any()


def test_write_nonfinite():
    x = torch.randn(4, 1, 64, device="cuda")
    x[0, 0, 3], x[1, 0, 40], x[2, 0, 5] = math.nan, math.inf, -math.inf
    x[3, 0, :32] = math.inf
    cache = QuantKVCache(1, 4, num_kv_heads=1, head_dim=64)
    rows = KVRows([0], [4])
    cache.write(x, torch.zeros_like(x), rows)
    with pytest.raises(KVCacheError, match="NaN or infinity"):
        cache.check_status()
    k, v = cache.read(rows, dtype=torch.float32)
    assert torch.equal(k, held(x, 4).float()) and not v.any() and torch.isfinite(k).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_strides_and_alignment(dtype):
    """Rows from a fused projection's output (strided, offset by elements) and
    transposed layouts; read and attend into strided tensors."""
    g = torch.Generator(device="cuda").manual_seed(3)
    n, hk, d = 21, 2, 64
    wide = torch.randn(n, 3 * hk * d + 1, generator=g, device="cuda").to(dtype)
    cache = QuantKVCache(1, 64, num_kv_heads=hk, head_dim=d)
    rows = KVRows([11], [n])
    for off in (0, 1):
        k = wide[:, off:off + hk * d].unflatten(1, (hk, d))
        v = wide[:, off + hk * d:off + 2 * hk * d].unflatten(1, (hk, d)).transpose(0, 1).contiguous().transpose(0, 1)
        q = wide[:, off + 2 * hk * d:off + 3 * hk * d].unflatten(1, (hk, d))
        cache.write(k, v, rows)
        out = torch.full((n, hk * d * 2 + 3), 7.0, dtype=dtype, device="cuda")
        kr, vr = out[:, off:off + hk * d].unflatten(1, (hk, d)), out[:, -hk * d:].unflatten(1, (hk, d))
        cache.read(rows, out=(kr, vr))
        assert torch.equal(kr, held(k, 4).float().to(dtype)) and torch.equal(vr, held(v, 4).float().to(dtype))
        rest = torch.ones(out.shape[1], dtype=torch.bool)
        rest[off:off + hk * d] = False
        rest[-hk * d:] = False
        assert (out[:, rest.cuda()] == 7.0).all()
        wide_out = torch.full((n, hk * d + 2), 7.0, dtype=dtype, device="cuda")
        got = wide_out[:, off:off + hk * d].unflatten(1, (hk, d))
        assert cache.attend(q, rows, out=got) is got
        same = cache.attend(q.contiguous(), rows)
        assert torch.equal(got, same)
        assert (wide_out[:, off + hk * d:] == 7.0).all() and (wide_out[:, :off] == 7.0).all()
    cache.check_status()


# ------------------------------------------------------------------- attend
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d,hk,ratio", [(128, 2, 2), (128, 1, 1), (64, 3, 4), (128, 1, 7), (64, 1, 16)])
def test_attend_single_rows(dtype, bits, d, hk, ratio):
    """One row a sequence at lengths around every tile size."""
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300, 1000, 2049]
    f = Filled(lens, hk=hk, d=d, bits=bits, seed=d + ratio)
    q = (1.5 * torch.randn(len(lens), hk * ratio, d, generator=f.gen, device="cuda")).to(dtype)
    got = f.cache.attend(q, KVRows([n - 1 for n in lens]))
    f.check(got, q, [(i, n - 1, 1) for i, n in enumerate(lens)])
    f.cache.check_status()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d,hk,ratio", [(128, 2, 2), (64, 1, 8), (128, 1, 1), (64, 2, 3), (128, 1, 7), (64, 1, 16)])
@pytest.mark.parametrize("counts", [(2, 1, 3), (5, 0, 9), (33, 17, 1), (64, 65, 63), (1, 200, 0), (257, 130, 2)], ids=str)
def test_attend_segments(dtype, bits, d, hk, ratio, counts):
    """Segments of several rows: chunks at positions off the tile borders, a
    fresh prompt, an empty segment, sequences in another order, one of them
    twice."""
    lens = [300, 411, 700, 5]
    f = Filled(lens, hk=hk, d=d, bits=bits, seed=sum(counts))
    segs = [(2, 131, counts[0]), (1, 0, counts[1]), (2, 700 - counts[2], counts[2]), (3, 4, 1)]
    rows = KVRows([s for _, s, _ in segs], [c for _, _, c in segs], [q for q, _, _ in segs])
    q = (1.5 * torch.randn(rows.rows, hk * ratio, d, generator=f.gen, device="cuda")).to(dtype)
    got = f.cache.attend(q, rows)
    f.check(got, q, segs)
    f.cache.check_status()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("hk,ratio", [(8, 2), (4, 13), (2, 16)], ids=str)
def test_single_rows_among_prompts(hk, ratio, dtype):
    """Blocks of few rows one after another and between full ones: whatever
    order a worker meets them in, no row takes another's query."""
    lens = [5, 60, 128, 129, 300, 957, 700]
    f = Filled(lens, hk=hk, seed=ratio)
    segs = []
    for i in range(60):
        s = i % 5
        segs.append((s, (37 * i) % lens[s], 1))
        if i % 20 == 7:
            segs.append((5, 15 * i, 249 if ratio == 13 else 130))
        if i % 20 == 15:
            segs.append((6, 3 * i, 33))
    q = torch.randn(sum(n for _, _, n in segs), hk * ratio, 128, generator=f.gen, device="cuda").to(dtype)
    rows = KVRows([a for _, a, _ in segs], [n for _, _, n in segs], [s for s, _, _ in segs])
    for _ in range(3):
        got = f.cache.attend(q, rows)
        f.cache.check_status()
        f.check(got, q, segs)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows", [1, 40, 150])
def test_attend_peaked_and_spread_scores(dtype, rows):
    """Scores up to several hundred (one position takes all) and all alike."""
    f = Filled([400], hk=1, d=128, seed=9)
    g = torch.randn(rows, 2, 128, generator=f.gen, device="cuda")
    segs = [(0, 400 - rows, rows)]
    for gain in (30.0, 1e-6):
        q = (gain * g).to(dtype)
        f.check(f.cache.attend(q, KVRows([400 - rows], [rows])), q, segs)
    q = g.to(dtype)
    f.check(f.cache.attend(q, KVRows([400 - rows], [rows]), scale=0.5), q, segs, scale=0.5)
    f.check(f.cache.attend(q, KVRows([400 - rows], [rows]), scale=-0.2), q, segs, scale=-0.2)
    q = torch.zeros_like(q)
    f.check(f.cache.attend(q, KVRows([400 - rows], [rows])), q, segs)


@pytest.mark.parametrize("rows", [1, 3, 100])
@pytest.mark.parametrize("gain", [1e-9, 3e4, 1e12])
def test_attend_small_and_large_values(rows, gain):
    """V of small and large magnitude (fp32 q and out: nothing saturates), and
    sequences that mix both."""
    f = Filled([300], hk=1, d=128, dtype=torch.float32, seed=4, v_gain=gain)
    q = torch.randn(rows, 2, 128, generator=f.gen, device="cuda")
    f.check(f.cache.attend(q, KVRows([300 - rows], [rows])), q, [(0, 300 - rows, rows)])
    f.v[0][::3] *= 1e-6
    f.v[0][7] = 0.0
    f.cache.write(f.k[0], f.v[0], KVRows([0], [300]))
    f.check(f.cache.attend(q, KVRows([300 - rows], [rows])), q, [(0, 300 - rows, rows)])


@pytest.mark.parametrize("rows", [1, 4, 90])
@pytest.mark.parametrize("bits", [4, 8])
def test_attend_ignores_what_a_row_does_not_see(rows, bits):
    """Rows past the limit hold garbage, NaN scales among it; the outputs do
    not change by a bit.  A NaN query spoils its own row alone."""
    n = 150
    f = Filled([n], hk=2, d=128, bits=bits, max_seq_len=400, seed=6)
    c = f.cache
    q = torch.randn(rows, 4, 128, generator=f.gen, device="cuda", dtype=torch.bfloat16)
    r = KVRows([n - rows], [rows])
    clean = c.attend(q, r)
    c.k_codes[:, :, :, n:] = 0xA5
    c.v_codes[:, :, :, n:] = 0x3C
    c.k_scales[:, :, :, n:] = math.nan
    c.v_scales[:, :, :, n::2] = math.nan
    c.v_scales[:, :, :, n + 1::2] = math.inf
    assert torch.equal(c.attend(q, r), clean)
    if rows > 1:
        q2 = q.clone()
        q2[1, 2, 5] = math.nan
        got = c.attend(q2, r)
        assert got[1, 2].isnan().all()
        got[1, 2] = clean[1, 2]
        assert torch.equal(got, clean)


@pytest.mark.parametrize("rows", [1, 3, 80])
def test_bad_rows_and_rows_of_no_segment(rows):
    """Device-side rows out of range: reported, zeros out, nothing written;
    rows past the last segment are left as they were."""
    f = Filled([100, 100], hk=1, d=64, seed=8)
    c = f.cache
    dev = dict(dtype=torch.int32, device="cuda")
    n = 4 * rows + 2
    start = torch.tensor([100 - rows, 99 - rows + 2, -1, 0], **dev)  # the second runs past the end
    seq = torch.tensor([0, 1, 0, 2], **dev)
    offs = torch.tensor([1, 1 + rows, 1 + 2 * rows, 1 + 3 * rows, 1 + 4 * rows], **dev)
    r = KVRows.from_tensors(start, offs, seq, rows=n, max_rows=rows)
    q = torch.randn(n, 2, 64, device="cuda", dtype=torch.bfloat16)
    out = torch.full_like(q, 5.0)
    c.attend(q, r, out=out)
    with pytest.raises(KVCacheError, match="out of range"):
        c.check_status()
    assert (out[0] == 5.0).all() and (out[-1] == 5.0).all()
    f.check(out[1:1 + rows], q[1:1 + rows], [(0, 100 - rows, rows)])
    if rows > 1:
        f.check(out[1 + rows:2 * rows], q[1 + rows:2 * rows], [(1, 101 - rows, rows - 1)])
    assert not out[2 * rows].any() and not out[1 + 2 * rows:1 + 4 * rows].any()
    k = torch.full((n, 1, 64), 3.0, device="cuda")
    kr, vr = k.clone(), k.clone()
    c.read(r, out=(kr, vr))
    with pytest.raises(KVCacheError, match="out of range"):
        c.check_status()
    assert (kr[0] == 3.0).all() and (vr[-1] == 3.0).all() and not kr[2 * rows:1 + 4 * rows].any()
    before = c.k_codes.clone()
    c.write(k, k, r)
    with pytest.raises(KVCacheError, match="out of range"):
        c.check_status()
    changed = (c.k_codes != before).any(-1)[:, 0, 0].nonzero().tolist()
    want = [[0, p] for p in range(100 - rows, 100)] + [[1, p] for p in range(101 - rows, 100)]
    assert changed == want
    # more rows in a segment than the caller allowed for
    if rows > 1:
        short = KVRows.from_tensors(start, offs, seq, rows=n, max_rows=rows - 1)
        out.fill_(5.0)
        c.attend(q, short, out=out)
        with pytest.raises(KVCacheError, match="out of range"):
            c.check_status()
        assert not out[rows].any()


def test_wild_offsets_stay_inside():
    """row_offsets that decrease or point outside reach no row outside the
    tensors (the neighbours keep their values)."""
    f = Filled([50, 50], hk=1, d=64, seed=1)
    dev = dict(dtype=torch.int32, device="cuda")
    for o in ([5, -7, 900], [-3, 2, 1 << 30], [8, 3, 8], [0, 2**31 - 1, -2**31]):
        r = KVRows.from_tensors(torch.tensor([10, 20], **dev), torch.tensor(o, **dev), rows=8, max_rows=8)
        wide = torch.full((24, 2, 64), 5.0, device="cuda", dtype=torch.bfloat16)
        f.cache.attend(torch.randn_like(wide[8:16]), r, out=wide[8:16])
        f.cache.read(r, out=(wide[8:16, :1], wide[8:16, 1:]))
        torch.cuda.synchronize()
        assert (wide[:8] == 5.0).all() and (wide[16:] == 5.0).all()
        f.cache.status.zero_()


@pytest.mark.parametrize("rows", [1, 100])
def test_segments_without_rows(rows):
    """Device offsets that give no segment a row: nothing is read or written."""
    f = Filled([50, 50], hk=1, d=64, seed=1)
    dev = dict(dtype=torch.int32, device="cuda")
    r = KVRows.from_tensors(torch.tensor([10, 20], **dev), torch.zeros(3, **dev), rows=100, max_rows=min(rows, 50))
    q = torch.randn(100, 2, 64, device="cuda", dtype=torch.bfloat16)
    out = torch.full_like(q, 5.0)
    f.cache.attend(q, r, out=out)
    assert (out == 5.0).all() and not f.cache.attend(q, r).any()
    before = f.cache.k_codes.clone()
    f.cache.write(out[:, :1], out[:, :1], r)
    assert torch.equal(f.cache.k_codes, before) and not f.cache.read(r)[0].any()
    f.cache.check_status()


@pytest.mark.parametrize("rows", [1, 3, 90])
def test_attend_in_place(rows):
    """out may be q itself."""
    f = Filled([600], hk=2, d=128, seed=21)
    q = torch.randn(rows, 4, 128, generator=f.gen, device="cuda", dtype=torch.bfloat16)
    r = KVRows([600 - rows], [rows])
    want = f.cache.attend(q, r)
    assert torch.equal(f.cache.attend(q, r, out=q), want)


def test_offsets_past_32_bits():
    """A cache of several GB: the last sequence's last positions."""
    n, seqs = 131072, 36
    c = QuantKVCache(seqs, n, num_kv_heads=8, head_dim=128, bits=8)
    assert c.k_codes.numel() > 2**32
    g = torch.Generator(device="cuda").manual_seed(2)
    k = torch.randn(n, 8, 128, generator=g, device="cuda", dtype=torch.bfloat16)
    v = torch.randn(n, 8, 128, generator=g, device="cuda", dtype=torch.bfloat16)
    c.write(k, v, KVRows([0], [n], [seqs - 1]))
    rows = KVRows([n - 5], [5], [seqs - 1])
    kr, vr = c.read(rows, dtype=torch.float32)
    assert torch.equal(kr, held(k[-5:], 8).float()) and torch.equal(vr, held(v[-5:], 8).float())
    assert not c.k_codes[:seqs - 1, :, :, -8:].any()
    q = torch.randn(5, 8, 128, generator=g, device="cuda", dtype=torch.bfloat16)
    got = c.attend(q, rows)
    for h in (0, 7):
        kh, vh = held(k[:, h:h + 1], 8), held(v[:, h:h + 1], 8)
        check_attend(got[:, h:h + 1], q[:, h:h + 1], kh, vh, [n - 4 + i for i in range(5)], 8,
                     1 / math.sqrt(128))


def test_repeatable_and_independent_of_neighbours():
    """Equal calls give equal bits, on any stream; a row's output does not
    depend on which sequences share the call beyond the order of sums."""
    f = Filled([700, 64, 333, 1], hk=4, d=128, seed=12)
    q = torch.randn(4, 8, 128, generator=f.gen, device="cuda", dtype=torch.float32)
    rows = KVRows([699, 63, 332, 0])
    first = f.cache.attend(q, rows)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:  # three calls in flight at once
        with torch.cuda.stream(s):
            outs.append([f.cache.attend(q, rows) for _ in range(5)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for group in outs for o in group)
    f.check(first, q, [(0, 699, 1), (1, 63, 1), (2, 332, 1), (3, 0, 1)])


def test_graph_replay_with_moving_positions():
    """write + attend captured once and replayed while the rows' tensors
    advance; two graphs of one cache replayed in turn."""
    hk, d, steps = 2, 128, 40
    c = QuantKVCache(2, 128, num_kv_heads=hk, head_dim=d, bits=4)
    g = torch.Generator(device="cuda").manual_seed(5)
    k = torch.randn(steps, 2, hk, d, generator=g, device="cuda", dtype=torch.bfloat16)
    v = torch.randn(steps, 2, hk, d, generator=g, device="cuda", dtype=torch.bfloat16)
    q = torch.randn(steps, 2, 2 * hk, d, generator=g, device="cuda", dtype=torch.bfloat16)
    start = torch.zeros(2, dtype=torch.int32, device="cuda")
    rows = KVRows.from_tensors(start)
    kb, vb, qb = k[0].clone(), v[0].clone(), q[0].clone()
    out = torch.empty_like(qb)
    c.write(kb, vb, rows)
    c.attend(qb, rows, out=out)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            c.write(kb, vb, rows)
            c.attend(qb, rows, out=out)
            start.add_(1)
        graphs.append(gr)
    start.zero_()
    c.reset()
    for t in range(steps):
        kb.copy_(k[t]), vb.copy_(v[t]), qb.copy_(q[t])
        graphs[t % 2].replay()
        for s in range(2):
            kh, vh = held(k[:t + 1, s], 4), held(v[:t + 1, s], 4)
            check_attend(out[s:s + 1], q[t, s:s + 1], kh, vh, [t + 1], 4, 1 / math.sqrt(d))
    c.check_status()


def test_prompt_then_steps_together():
    """The run that a serving loop makes: a ragged batch of prompts written
    and attended, then single-row steps, every output against the formulas."""
    hk, d = 2, 64
    lens = [70, 1, 130]
    c = QuantKVCache(3, 200, num_layers=2, num_kv_heads=hk, head_dim=d, bits=8)
    g = torch.Generator(device="cuda").manual_seed(7)
    ks, vs = [[] for _ in lens], [[] for _ in lens]

    def feed(counts, starts):
        rows = KVRows(starts, counts)
        k = torch.randn(rows.rows, hk, d, generator=g, device="cuda", dtype=torch.float16)
        v = torch.randn(rows.rows, hk, d, generator=g, device="cuda", dtype=torch.float16)
        q = torch.randn(rows.rows, 3 * hk, d, generator=g, device="cuda", dtype=torch.float16)
        c.write(k, v, rows, layer=1)
        out = c.attend(q, rows, layer=1)
        r = 0
        for s, n in enumerate(counts):
            ks[s].append(k[r:r + n])
            vs[s].append(v[r:r + n])
            kh, vh = held(torch.cat(ks[s]), 8), held(torch.cat(vs[s]), 8)
            check_attend(out[r:r + n], q[r:r + n], kh, vh, [starts[s] + i + 1 for i in range(n)], 8,
                         1 / math.sqrt(d))
            r += n

    feed(lens, [0, 0, 0])
    for t in range(4):
        feed([1, 1, 1], [n + t for n in lens])
    c.check_status()


def test_refusals_on_the_device():
    c = QuantKVCache(1, 32, num_kv_heads=2, head_dim=64)
    rows = KVRows([0], [4])
    x = torch.zeros(4, 2, 64, device="cuda")
    for bad in (x.double(), x.int(), x.cpu(), x[:, :1], x.transpose(1, 2).contiguous().transpose(1, 2)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            c.write(bad, x if bad.is_cuda else bad, rows)
    with pytest.raises(RuntimeError):
        c.write(x, x.half(), rows)
    with pytest.raises(RuntimeError):
        c.read(rows, out=(x, x[:1].expand(4, 2, 64)))
    with pytest.raises(RuntimeError):
        c.attend(x, rows, out=x[:1].expand(4, 2, 64))
    with pytest.raises(RuntimeError):
        c.attend(x, KVRows.from_tensors(torch.zeros(4, dtype=torch.int64, device="cuda")))
    with pytest.raises(RuntimeError):
        c.attend(x, KVRows.from_tensors(torch.zeros(4, dtype=torch.int32)))
    with pytest.raises(RuntimeError):  # offsets of another length
        c.attend(x, KVRows.from_tensors(torch.zeros(2, dtype=torch.int32, device="cuda"),
                                        torch.zeros(2, dtype=torch.int32, device="cuda"), rows=4, max_rows=4))
    empty = x[:0]
    c.write(empty, empty, KVRows([0], [0]))
    assert c.attend(empty, KVRows([0], [0])).shape == (0, 2, 64)
    c.check_status()
