"""4-bit KV cache operators against 64 bits, with bounds that follow their arithmetic term by term.

A stored row stands for s n + b per element; hat(x) = |s| n + |b| bounds what its parts sum up to.  Half steps:
bf16 2^-8, fp16 2^-11, fp32 2^-24.

* score: the integers, the queries and the key offsets enter the tensor cores exactly, or as 22 bits and more (offsets of
  the chunk form: two fp16 terms; elements 2^-22 below the largest K are lost).  What is left are fp32 sums: at most
  eight matrix steps of 16 terms per row, each of which may lose 17 last places of the largest partial sum, and ten
  roundings after them, (8 * 17 + 10) 2^-24 < 2^-16.8 of the magnitudes' sum: e = 2^-16.5 |scale| (sum_d |q_d| hat(k_jd)) +
  2^-21 |scale| max|k| sum_d |q_d|, the largest over the row's keys, and 2^-21 for the power of two itself.
* probability: a factor exp(2 e).
* output: p s or p, and V in the chunk form, are rounded to 11 bits: sum_j p_j hat(v_j) (2 * 2^-11 + expm1(2 e)), sums of
  the keys in fp32 (2^-13 of the same sum covers chains of 2048 additions), 2^-21 of the largest |v|, and the
  final rounding 2^-8 |out|.  V below 2^-90 is held to 2^-111 instead: the powers of two that bring V into fp16 end at 2^98
  (chunks: half of the last place 2^-24 is 2^-123) and p s is held against 2^-79 at least (2^-25 of 2^-79 2^-11, 15 times:
  2^-111), and bf16 itself ends at 2^-133.
* log-sum-exp: e, and 2^-13 relative of the sum (2^-13 absolute of its logarithm), 2^-22 |lse|.
* weight of a key: factors exp(2 e) of its probabilities and 2^-12 of them (the log-sum-exp's sum), fp32 sums with what
  was there: 2^-20 (1 + |mass|).
"""
from fractions import Fraction

import pytest

from test_gpu_kv4 import CASES, Cache, _append, _attend, _dev, _evict, _filled, _kept, _quantize64, _rand

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


def _parts(c, which):
    """float64 values and hat magnitudes [B, H, max_pos, D] of the stored rows, on the GPU."""
    torch = _torch()
    w, s, b = c.t[3 * which:3 * which + 3]
    s, b = (t.view(torch.bfloat16).double().repeat_interleave(64, -1) for t in (s, b))
    n = ((w.long()[..., None] >> torch.arange(0, 32, 4, device=w.device)) & 15).reshape(s.shape).double()
    return s * n + b, s.abs() * n + b.abs()


def _bounds(c, x, off, n, causal=True, scale=None, leave_out=None):
    """Per sequence b: (out, its bound [rows, Hq, D], lse, its bound [rows, Hq], weights, their bound [H, keys]) of its n[b]
    rows behind off[b] positions.  leave_out: a range of keys that the result (not the bounds) goes without."""
    torch = _torch()
    B, S, Hq, D = x.shape
    H, G = c.H, Hq // c.H
    scale = D ** -0.5 if scale is None else scale
    (K, Kh), (V, Vh) = _parts(c, 0), _parts(c, 1)
    res = []
    for b in range(B):
        r, T = n[b], off[b] + n[b]
        o, to, z, tz, m, tm = [], [], [], [], [], []
        hide = torch.zeros(r, T, dtype=torch.bool, device=x.device)
        if causal:
            hide = torch.arange(T, device=x.device)[None] > torch.arange(off[b], T, device=x.device)[:, None]
        gone = hide.clone()
        if leave_out:
            gone[:, leave_out[0]:leave_out[1]] = True
        for h in range(H):
            k, kh, v, vh = (t[b, h, :T] for t in (K, Kh, V, Vh))
            q = x[b, :r, h * G:(h + 1) * G].double()
            s = scale * torch.einsum("igd,jd->igj", q, k)
            e = 2.0 ** -16.5 * abs(scale) * torch.einsum("igd,jd->igj", q.abs(), kh) + \
                2.0 ** -21 * (1 + abs(scale) * k.abs().max() * q.abs().sum(-1, keepdim=True))
            e = e.masked_fill(hide[:, None], 0).amax(-1)
            zf = torch.logsumexp(s.masked_fill(hide[:, None], -float("inf")), -1)
            pf = torch.exp(s.masked_fill(hide[:, None], -float("inf")) - zf[..., None])
            s = s.masked_fill(gone[:, None], -float("inf"))
            zz = torch.logsumexp(s, -1)
            p = torch.exp(s - zz[..., None])
            out = torch.einsum("igj,jd->igd", p, v)
            o.append(out)
            to.append(torch.einsum("igj,jd->igd", pf, vh) * (2.0 ** -10 + 2.0 ** -13 + torch.expm1(2 * e)[..., None])
                      + 2.0 ** -21 * v.abs().max().clamp(min=2.0 ** -90) + 2.0 ** -8 * torch.einsum("igj,jd->igd", pf, v).abs())
            z.append(zz)
            tz.append(e + 2.0 ** -13 + 2.0 ** -22 * zf.abs())
            m.append(p.sum((0, 1)))
            tm.append((pf * (torch.expm1(2 * e)[..., None] + 2.0 ** -12)).sum((0, 1)) + 2.0 ** -20 * (1 + pf.sum((0, 1))))
        res.append((torch.cat(o, 1), torch.cat(to, 1), torch.cat(z, 1), torch.cat(tz, 1), torch.stack(m), torch.stack(tm)))
    return res


# Euclidean norm of a row's error, relative to its output's, where V is independent of the probabilities: the roundings are
# independent too, so those of p and v add up to at most 2 * 2^-11 sqrt(sum p^2 hat(v)^2) against sqrt(sum p^2 v^2), with hat(v)
# at most five times v in the mean of normal rows: 5 * 2^-10, and 2^-8 for the final rounding; together below 2^-6.7.
NORM = 2.0 ** -6


def _check(c, x, off, n=None, causal=True, scale=None, mass=True, norm=None, **kw):
    """The call's output, log-sum-exp and weights lie within the bounds."""
    torch = _torch()
    n = [x.shape[1]] * x.shape[0] if n is None else n
    m = torch.zeros(c.B, c.H, c.max_pos, device=x.device) if mass else None
    out, lse = _attend(c, x, _dev(off), _dev(n), causal=causal, scale=scale, mass=m, **kw)
    for b, (o, to, z, tz, w, tw) in enumerate(_bounds(c, x, off, n, causal, scale)):
        d = (out[b, :n[b]].double() - o).abs()
        assert (d <= to).all(), (b, (d / to).max())
        assert norm is None or (d.norm(dim=-1) <= norm * o.norm(dim=-1)).all(), (b, (d.norm(dim=-1) / o.norm(dim=-1)).max())
        d = (lse[b, :n[b]].double() - z).abs()
        assert (d <= tz).all(), (b, (d / tz).max())
        assert (out[b, n[b]:] == 0).all() and (lse[b, n[b]:] == -float("inf")).all()
        if mass:
            T = off[b] + n[b]
            d = (m[b, :, :T].double() - w).abs()
            assert (d <= tw).all(), (b, (d / tw).max())
            assert (m[b, :, T:] == 0).all()
    return out, lse, m


def _staircase(D, T, H=2):
    """Keys whose scores (base 2) rise by 9 in every 64 positions: position 64 r + 5 is at 9 (r + 1), the others of its 64 at 9 r,
    so that they hold a seventh of the weight.  Rows of +-7.5 s with s = m 2^-6, m <= 16, are stored exactly."""
    torch = _torch()
    c = Cache(1, H, (T + 15) // 16 * 16, D)
    r = torch.arange(T) // 64
    level = torch.where(torch.arange(T) % 64 == 5, r + 1, r).float()
    sign = torch.where(torch.arange(D) % 2 == 0, 1.0, -1.0)
    k = (level * 7.5 * 2.0 ** -6)[:, None, None] * sign
    assert level.max() <= 16
    _append(c, k[None].expand(1, T, H, D).contiguous().bfloat16().cuda(), _rand((1, T, H, D), 2).cuda(), _dev([0]))
    beta = 9.0 / (D * 7.5 * 2.0 ** -6 * D ** -0.5 * 1.4426950408889634)
    return c, beta * sign


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,G", [(1, 2), (20, 1), (70, 1), (90, 2), (64, 4)])
def test_scores_that_rise_in_both_halves_of_every_tile(S, G, D):
    """The running maximum moves in each 64 keys, in the first tile and in later ones: what has been summed is scaled twice a tile."""
    torch = _torch()
    c, u = _staircase(D, 960)
    x = u * (1 + 0.002 * torch.arange(S * 2 * G).reshape(1, S, 2 * G, 1) / (S * 2 * G))
    x = (x + 0.01 * _rand((1, S, 2 * G, D), 5).float()).bfloat16().cuda()
    _check(c, x, [960 - S], mass=False)
    _check(c, x, [960 - S], mass=False, causal=False)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,Hq,Hkv,T", [(64, 2, 2, 700), (300, 8, 2, 300), (600, 4, 1, 1500), (1024, 4, 1, 1024)])
def test_weights_of_long_chunks(S, Hq, Hkv, T, D):
    """One to 32 tiles of columns, whose tables are reused, with queries of very different size from column to column; every run
    gives the same bits."""
    torch = _torch()
    c = _filled(2, Hkv, T, D, outliers=False)
    x = _rand((2, S, Hq, D), 3).float()
    x = (x * torch.exp2(-6 * torch.rand(2, S, Hq, 1, generator=torch.Generator().manual_seed(4)))).bfloat16().cuda()
    off, n = [T - S, 0], [S, S - S // 3]
    _, _, m = _check(c, x, off, n)
    _check(c, x, off, n, causal=False)
    for _ in range(6):
        again = torch.zeros_like(m)
        _attend(c, x, _dev(off), _dev(n), mass=again)
        assert torch.equal(again, m)


def _words(q, D):
    """uint32 words (as int32) of 4-bit integers [..., D]."""
    torch = _torch()
    w = (q.long().reshape(*q.shape[:-1], D // 8, 8) << torch.arange(0, 32, 4)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,shift", [(5, 0), (700, 0), (700, 3)])
def test_append_of_groups_wider_than_fp32(S, shift, D):
    """Groups of large magnitudes only, max - min past the fp32 range: the words of the exact quotients."""
    torch = _torch()
    g = torch.Generator().manual_seed(S)
    kinds = torch.tensor([[3e38, -3e38, 1e38, -1e38, 2e38, -2e38, 5e37, -5e37], [3e38, -3e38] * 4, [2e38, -2e38, 2e38, -1.9e38] * 2,
                          [3.38e38, -3.38e38, 1e34, -1e34] * 2]).bfloat16()
    x = kinds[torch.randint(0, 4, (1, S, 8, D // 8), generator=g)].reshape(1, S, 8, D)  # a thread's eight values each
    x[0, ::3, ::2] = (x[0, ::3, ::2].float() * (0.5 + torch.rand(x[0, ::3, ::2].shape, generator=g))).clamp(-3.38e38, 3.38e38).bfloat16()
    c = Cache(1, 8, 768, D)
    y = torch.empty(1, S, 8, D + shift, dtype=torch.bfloat16)[..., shift:]
    y.copy_(x)
    k = torch.empty_strided(y.shape, (S * 8 * (D + shift), 8 * (D + shift), D + shift, 1), dtype=torch.bfloat16, device="cuda")
    k.copy_(x)
    _append(c, k, k, _dev([0]))
    q, s, z = _quantize64(x.double().transpose(1, 2))
    assert torch.isfinite(s).all()
    for which in (0, 1):
        assert torch.equal(c.t[3 * which][:, :, :S].cpu(), _words(q, D))
        assert torch.equal(c.t[3 * which + 1][:, :, :S].cpu().view(torch.bfloat16).double(), s)
        assert torch.equal(c.t[3 * which + 2][:, :, :S].cpu().view(torch.bfloat16).double(), z)


def _nearest(x, bias, scale):
    """The integer nearest to the exact (x - bias) / scale, ties to even, in 0..15: rational arithmetic."""
    f = (Fraction(float(x)) - Fraction(float(bias))) / Fraction(float(scale))
    return max(0, min(15, round(f)))  # round() of a Fraction takes ties to even


@pytest.mark.parametrize("tiny", [2.0 ** -30, 2.0 ** -60, 2.0 ** -110, 2.0 ** -126])
def test_append_of_quotients_a_hair_from_a_half(tiny):
    """(x - bias) / scale next to n + 1/2 by far less than 64 bits of floating point hold: small x beside a bias of
    (n + 1/2) scale, and x of (n + 1/2) scale beside a small bias."""
    torch = _torch()
    rows = []
    for scale in (2.0, 1.5, 2.0 ** 20, 23 * 2.0 ** -9):
        for n in range(6):
            r = torch.zeros(64)
            r[0] = -(n + 0.5) * scale
            r[1] = (15 - n - 0.5) * scale
            r[2:22] = torch.tensor([tiny, -tiny, 2 * tiny, -3 * tiny, 0.0] * 4)
            rows.append(r)
        for sign in (1, -1):
            r = torch.zeros(64)
            r[0] = -tiny
            r[1] = 15 * scale
            r[2:17] = (torch.arange(15) + 0.5) * scale
            rows.append(r * sign)
    x = torch.stack(rows).bfloat16()[None, :, None]  # [1, rows, 1, 64]
    S = x.shape[1]
    c = Cache(1, 1, 64, 64)
    _append(c, x.cuda(), x.cuda(), _dev([0]))
    w = c.t[0][0, 0, :S].cpu().long()
    got = ((w[..., None] >> torch.arange(0, 32, 4)) & 15).reshape(S, 64)
    s = c.t[1][0, 0, :S, 0].cpu().view(torch.bfloat16)
    z = c.t[2][0, 0, :S, 0].cpu().view(torch.bfloat16)
    for i in range(S):
        assert float(z[i]) == float(x[0, i, 0].min())
        want = [_nearest(v, z[i], s[i]) for v in x[0, i, 0]]
        assert got[i].tolist() == want, (i, float(s[i]))


@pytest.mark.parametrize("T", [200, 9000])
@pytest.mark.parametrize("S,G,row", [(2, 1, 0), (5, 2, 1), (5, 3, 3), (8, 2, 4), (20, 1, 7), (9, 6, 2), (70, 1, 3), (100, 2, 64)])
def test_weights_beside_a_nan_query(S, G, row, T):
    """A NaN query makes the weights of the keys that its row sees NaN; the keys behind them have the other rows' weights."""
    torch = _torch()
    c = _filled(1, 2, T, 64, outliers=False)
    x = _rand((1, S, 2 * G, 64), 3)
    off = T - S
    _, _, _, _, want, tol = _bounds(c, x.cuda(), [off], [S])[0]
    x[0, row, 0, 7] = float("nan")  # a head of kv head 0
    m = torch.zeros(1, 2, c.max_pos, device="cuda")
    out, lse = _attend(c, x.cuda(), _dev([off]), mass=m)
    seen = off + row + 1
    assert torch.isnan(m[0, 0, :seen]).all()
    assert ((m[0, 0, seen:T].double() - want[0, seen:]).abs() <= tol[0, seen:]).all()
    assert ((m[0, 1, :T].double() - want[1]).abs() <= tol[1]).all()
    nan = torch.isnan(out).all(-1)[0]
    assert nan[row, 0] and int(nan.sum()) == 1 and int(torch.isnan(lse).sum()) == 1


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("S,G,T,at", [(1, 4, 300, 299), (5, 4, 300, 297), (20, 2, 300, 290), (90, 1, 300, 250), (90, 2, 300, 10),
                                      (70, 2, 9000, 8960), (200, 2, 1500, 1301), (300, 1, 300, 0), (300, 1, 300, 260)])
@pytest.mark.parametrize("D", [64, 128])
def test_a_value_that_is_not_finite_leaves_sums_and_weights(S, G, T, at, D, bad):
    """Log-sum-exp and weights come from K alone: a V that is not finite changes neither, and only the outputs that see it."""
    torch = _torch()
    c = _filled(1, 1, T, D, outliers=False)
    x = _rand((1, S, G, D), 3).cuda()
    off = T - S
    want, to, z, tz, w, tw = _bounds(c, x, [off], [S])[0]
    c.t[4][0, 0, at, 0] = int(torch.tensor(float("nan")).bfloat16().view(torch.int16)) if bad != bad else c.t[4][0, 0, at, 0]
    c.t[5][0, 0, at, 0] = int(torch.tensor(bad).bfloat16().view(torch.int16))
    m = torch.zeros(1, 1, c.max_pos, device="cuda")
    out, lse = _attend(c, x, _dev([off]), mass=m)
    assert ((lse[0].double() - z).abs() <= tz).all()
    assert ((m[0, :, :T].double() - w).abs() <= tw).all()
    sees = torch.arange(S, device="cuda") + off >= at
    assert not torch.isfinite(out[0, sees][..., :64].float()).any()
    if bad != bad:
        assert torch.isnan(out[0, sees][..., :64]).all()
    assert ((out[0, ~sees].double() - want[~sees]).abs() <= to[~sees]).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("vmul", [1e-36, 1e-30, 1e29, 1e33, 3e36])
@pytest.mark.parametrize("S,G,T", [(64, 1, 6000), (64, 4, 2100)])
def test_split_chunks_of_very_large_and_small_values(S, G, T, vmul, D):
    """Values up to the end of bf16 where a chunk's keys are split over thread blocks: their partial sums stay finite."""
    torch = _torch()
    c = Cache(1, 1, (T + 63) // 64 * 64, D)
    v = (_rand((1, T, 1, D), 2).float() * vmul).bfloat16().cuda()
    v[0, T // 2:] *= 2.0 ** -10  # shares of different magnitude
    _append(c, _rand((1, T, 1, D), 1).cuda(), v, _dev([0]))
    x = _rand((1, S, G, D), 3).cuda()
    _check(c, x, [T - S])
    _check(c, x, [T - S], causal=False)


@pytest.mark.parametrize("value", [3e-38, 1.0, 1e6, 1e12, 1e25, 3e38])
@pytest.mark.parametrize("S,G,T", [(1, 4, 1), (1, 4, 40), (1, 4, 12000), (1, 16, 9000), (5, 2, 700), (20, 2, 9000), (90, 1, 700)])
def test_values_that_are_constant_in_every_group(S, G, T, value):
    """Scales of zero and biases of any size: the sums of biases stay in range, whichever keys come first."""
    torch = _torch()
    for kind in range(2):
        c = Cache(1, 2, (T + S + 63) // 64 * 64, 128)
        v = torch.full((1, T + S, 2, 128), value)
        v[..., 64:] *= -0.5
        if kind:  # zeros first, then rows of the value
            v[:, :(T + S) // 2] = 0.0
        _append(c, _rand((1, T + S, 2, 128), 1).cuda(), v.bfloat16().cuda(), _dev([0]))
        assert (c.t[4][:, :, :T + S] == 0).all()
        _check(c, _rand((1, S, 2 * G, 128), 3).cuda(), [T])


@pytest.mark.parametrize("inplace", [False, True])
def test_evict_takes_a_length_out_of_range_for_an_empty_sequence(inplace):
    """As the other operators do: nothing is moved or read, the new length is 0."""
    torch = _torch()
    src = _filled(6, 2, 128, 64, max_pos=128)
    dst = src if inplace else Cache(6, 2, 48, 64)
    ms = torch.rand(6, 2, 128, generator=torch.Generator().manual_seed(1)).cuda()
    md = ms if inplace else torch.full((6, 2, 48), 9.0, device="cuda")
    before, m0, source = dst.bits(), md.clone(), ms.clone()
    lens = [-1, 129, -2 ** 31, 2 ** 31 - 1, 128, 20]
    index, new = _dev([[[77] * 40] * 2] * 6), _dev([-5] * 6)
    _evict(src, dst, ms, md, _dev(lens), new, 40, 8, index)
    assert new.tolist() == [0, 0, 0, 0, 40, 20]
    assert (index[:4] == -1).all() and (index[4] >= 0).all()
    for t0, t1 in zip(before, dst.bits()):
        assert torch.equal(t0[:4], t1[:4])
    assert torch.equal(md[:4], m0[:4])
    for h in range(2):
        assert index[4, h].tolist() == _kept(source[4, h].cpu().double().numpy(), 128, 40, 8).tolist()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("B,Hq,Hkv,D,S,total", CASES)
def test_attention_within_its_arithmetic(B, Hq, Hkv, D, S, total, causal):
    c = _filled(B, Hkv, max(total), D, seed=S)
    x = _rand((B, S, Hq, D), 77 + S, 1.5).cuda()
    _check(c, x, [t - S for t in total], causal=causal)


@pytest.mark.parametrize("S,Hq,Hkv,T,B,D", [
    (1, 32, 8, 20000, 1, 128), (1, 8, 1, 9000, 2, 128), (1, 16, 4, 700, 40, 128), (16, 16, 1, 4000, 1, 128), (300, 4, 1, 3000, 1, 128),
    (1, 16, 1, 9000, 2, 128), (5, 8, 2, 9001, 1, 128), (5, 8, 2, 5000, 3, 64), (1, 6, 1, 12345, 1, 64), (1, 64, 1, 3001, 2, 128),
    (130, 2, 1, 4111, 2, 64), (40, 8, 2, 2500, 3, 128), (700, 2, 1, 701, 1, 128), (5, 32, 8, 9000, 2, 64), (15, 3, 1, 6001, 2, 128)])
def test_long_attention_within_its_arithmetic(S, Hq, Hkv, T, B, D):
    """Keys split over thread blocks, clusters and column blocks: a share that is lost, scaled or joined wrongly is outside the
    bounds (see test_kv4_bounds_cpu.py)."""
    c = _filled(B, Hkv, T, D, outliers=False)
    total = [T] + [max(S, T * (i + 1) // (B + 1) + i % 7) for i in range(B - 1)]
    x = _rand((B, S, Hq, D), 12, 1.5).cuda()
    _check(c, x, [t - S for t in total], norm=NORM if min(total) - S > 64 else None)


@pytest.mark.parametrize("scale", [1e25, 1e31, 1.0e36])  # probabilities below 2^-136 scale of the largest may be lost: 2^-16
@pytest.mark.parametrize("S,G,T,D", [(1, 4, 200, 128), (1, 4, 9000, 128), (1, 16, 200, 64), (5, 2, 230, 64), (20, 1, 260, 128), (90, 1, 1200, 128)])
def test_a_very_large_value_scale_leaves_sums_and_weights(S, G, T, D, scale):
    """One key at 2^14 times the weight of each other, which together weigh half of it or less, and one very large
    value scale: log-sum-exp and weights come from K alone; the rows that do not see that key keep their outputs
    where it is the last one (but for 2^-22 of its values)."""
    torch = _torch()
    c = Cache(1, 1, (T + 15) // 16 * 16, D)
    sign = torch.where(torch.arange(D) % 2 == 0, 1.0, -1.0)
    k = torch.zeros(1, T, 1, D)
    k[0, 3, 0] = 7.5 * 2.0 ** -3 * sign
    _append(c, k.bfloat16().cuda(), _rand((1, T, 1, D), 2).cuda(), _dev([0]))
    beta = 14.0 / (D * 7.5 * 2.0 ** -3 * D ** -0.5 * 1.4426950408889634)
    x = (beta * sign).expand(1, S, G, D).bfloat16().cuda()
    _, _, z, tz, w, tw = _bounds(c, x, [T - S], [S])[0]
    for at in (T - 1, 20):
        d = Cache(1, 1, c.max_pos, D)
        for t, u in zip(d.t, c.t):
            t.copy_(u)
        d.t[4][0, 0, at, 0] = int(torch.tensor(scale).bfloat16().view(torch.int16))
        m = torch.zeros(1, 1, c.max_pos, device="cuda")
        out, lse = _attend(d, x, _dev([T - S]), mass=m)
        assert ((lse[0].double() - z).abs() <= tz).all(), (at, (lse[0].double() - z).abs().max())
        assert ((m[0, :, :T].double() - w).abs() <= tw).all(), at
        _, to, _, _, _, _ = _bounds(d, x, [T - S], [S])[0]
        o = _bounds(d, x, [T - S], [S])[0][0]
        vmax = 2.0 ** -21 * 31 * scale  # the chunk form's and the hidden key's part
        assert ((out[0].double() - o).abs() <= to + vmax).all(), at
