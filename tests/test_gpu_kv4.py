"""4-bit KV cache operators against plain implementations in 64 bits.

Tolerances, from the arithmetic (half steps: bf16 2^-8, fp16 2^-11, fp32 2^-24):

* rows: a stored value q is the nearest integer to the exact quotient, so words,
  scales and biases are equal bit for bit; a value read back is one fp32 fma
  (relative 2^-24) rounded to bf16: the exact value rounded to bf16, or its
  neighbour where the fp32 rounding crossed a midpoint.
* attention: keys, values and probabilities may enter the tensor cores as fp16
  (relative 2^-11 each), sums are fp32.  A score is off by at most e = (2^-11 +
  2^-16) * |scale| * max_j sum_d |q_d k_jd|, a probability by a factor exp(2 e),
  the output by vmax * (2 * 2^-11 + exp(2 e) - 1) with vmax the largest |value|
  (a stored value is bias + scale q with |bias|, scale q <= 2 max(|bias|, |bias + 15 scale|),
  so vmax = 3 times that bound covers values summed in two parts), plus the
  final rounding 2^-8 |out|; lse by e + 2^-20 (1 + |lse|); a key's weight by the factor
  exp(2 e), plus fp32 sums.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

GARBAGE = 0x7FC0  # NaN as bf16: scales and biases of rows no sequence has


def _torch():
    import torch
    return torch


def _api():
    import qwen3_b200
    return qwen3_b200


def _quantize64(x):
    """float64 [..., D] of bf16 values -> (q int64 [..., D], scale, bias float64 [..., D / 64])."""
    torch = _torch()
    g = x.reshape(*x.shape[:-1], -1, 64)
    lo, hi = g.min(-1).values, g.max(-1).values
    bad = ~torch.isfinite(g).all(-1)
    scale = ((hi - lo) / 15).float().bfloat16().double()
    safe = torch.where(scale == 0, torch.ones_like(scale), scale)
    q = ((g - lo[..., None]) / safe[..., None]).round().clamp(0, 15)
    q = torch.where((scale == 0)[..., None], torch.zeros_like(q), q)
    q = torch.where(bad[..., None], torch.zeros_like(q), q)
    nan = torch.full_like(scale, float("nan"))
    return q.reshape(x.shape).long(), torch.where(bad, nan, scale), torch.where(bad, nan, lo)


class Cache:
    """A cache on the GPU whose rows past the stored ones hold NaN scales and set bits."""

    def __init__(self, B, H, max_pos, D, device="cuda:0"):
        torch = _torch()
        self.B, self.H, self.max_pos, self.D, self.device = B, H, max_pos, D, device
        self.t = []
        for _ in range(2):
            self.t.append(torch.full((B, H, max_pos, D // 8), -1, dtype=torch.int32, device=device))
            for _ in range(2):
                self.t.append(torch.full((B, H, max_pos, D // 64), GARBAGE, dtype=torch.int16, device=device))
        self.h = _api().Kv4(*[t.data_ptr() for t in self.t], B, H, max_pos, D)

    def bits(self):
        return [t.cpu().clone() for t in self.t]

    def values64(self, which):
        """float64 [B, H, max_pos, D] of the stored rows, on the CPU."""
        torch = _torch()
        w, s, b = [t.cpu() for t in self.t[3 * which:3 * which + 3]]
        s, b = s.view(torch.bfloat16).double(), b.view(torch.bfloat16).double()
        sh = torch.arange(0, 32, 4)
        q = ((w.long()[..., None] >> sh) & 15).reshape(self.B, self.H, self.max_pos, self.D).double()
        return q * s.repeat_interleave(64, -1) + b.repeat_interleave(64, -1)


def _dev(x, dtype=None):
    torch = _torch()
    return torch.as_tensor(x, dtype=dtype or torch.int32, device="cuda:0")


def _rand(shape, seed, scale=1.0, outliers=False):
    torch = _torch()
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * scale
    if outliers:
        x[..., 5] *= 20
        x[..., 40] += 7
    return x.bfloat16()


def _append(c, k, v, seq_len, n_new=None, strides=True, err=None):
    torch = _torch()
    _api().kv4_append(c.h, k.data_ptr(), v.data_ptr(), k.shape[1], seq_len.data_ptr(),
                      n_new_ptr=0 if n_new is None else n_new.data_ptr(),
                      k_strides=k.stride()[:3] if strides else None, v_strides=v.stride()[:3] if strides else None,
                      err_ptr=0 if err is None else err.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)


def _attend(c, x, seq_len, n_new=None, causal=True, scale=None, mass=None, out=None, err=None, scratch=None,
            want_lse=True):
    torch, q = _torch(), _api()
    B, S, Hq, D = x.shape
    if out is None:
        out = torch.full((B, S, Hq, D), 7.0, dtype=torch.bfloat16, device=x.device)
    lse = torch.full((B, S, Hq), 7.0, device=x.device) if want_lse else None
    n = q.kv4_attention_scratch_bytes(c.h, S, Hq)
    if scratch is None:
        scratch = torch.full((max(n, 16),), 0xFF, dtype=torch.uint8, device=x.device)
    q.kv4_attention(c.h, x.data_ptr(), out.data_ptr(), S, Hq, D ** -0.5 if scale is None else scale,
                    seq_len.data_ptr(), scratch.data_ptr(), scratch.numel(),
                    n_new_ptr=0 if n_new is None else n_new.data_ptr(), causal=causal,
                    lse_ptr=0 if lse is None else lse.data_ptr(), mass_ptr=0 if mass is None else mass.data_ptr(),
                    q_strides=x.stride()[:3], out_strides=out.stride()[:3],
                    err_ptr=0 if err is None else err.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    return out, lse


def _reference(c, x, seq_len, n_new, causal, scale, mass=None):
    """(out, lse, mass, score bound e, vmax) in 64 bits on the CPU; e and vmax per row."""
    torch = _torch()
    B, S, Hq, D = x.shape
    H, G = c.H, Hq // c.H
    K, V = c.values64(0), c.values64(1)
    X = x.cpu().double()
    out, lse = torch.zeros(B, S, Hq, D).double(), torch.full((B, S, Hq), -float("inf")).double()
    e, vm = torch.zeros(B, S, Hq).double(), torch.zeros(B, S, Hq).double()
    m = None if mass is None else mass.cpu().double().clone()
    em = None if mass is None else torch.zeros_like(m)
    for b in range(B):
        off = max(0, min(int(seq_len[b]), c.max_pos))
        n = min(S if n_new is None else max(0, min(int(n_new[b]), S)), c.max_pos - off)
        for i in range(n):
            vis = off + i + 1 if causal else off + n
            for h in range(H):
                k, v = K[b, h, :vis], V[b, h, :vis]
                qr = X[b, i, h * G:(h + 1) * G]
                s = scale * (qr @ k.T)
                z = torch.logsumexp(s, -1)
                p = torch.exp(s - z[:, None])
                out[b, i, h * G:(h + 1) * G] = p @ v
                lse[b, i, h * G:(h + 1) * G] = z
                bound = (2.0 ** -11 + 2.0 ** -16) * abs(scale) * (qr.abs() @ k.abs().T).max(-1).values
                e[b, i, h * G:(h + 1) * G] = bound
                vm[b, i, h * G:(h + 1) * G] = 3 * v.abs().max()
                if m is not None:
                    m[b, h, :vis] += p.sum(0)
                    em[b, h, :vis] += (p * torch.expm1(2 * bound)[:, None]).sum(0)
    return out, lse, m, em, e, vm


def _check_attention(c, x, seq_len, n_new=None, causal=True, scale=None, mass=False, **kw):
    torch = _torch()
    scale = x.shape[-1] ** -0.5 if scale is None else scale
    m0 = None
    if mass:
        g = torch.Generator().manual_seed(99)
        m0 = torch.rand(c.B, c.H, c.max_pos, generator=g).cuda()
    m = None if m0 is None else m0.clone()
    out, lse = _attend(c, x, seq_len, n_new, causal, scale, m, **kw)
    torch.cuda.synchronize()
    ro, rl, rm, em, e, vm = _reference(c, x, seq_len.cpu(), None if n_new is None else n_new.cpu(), causal, scale, m0)
    err = (out.cpu().double() - ro).abs()
    tol = vm[..., None] * (2.0 ** -10 + torch.expm1(2 * e)[..., None]) + 2.0 ** -8 * ro.abs()
    assert (err <= tol).all(), (err - tol).max()
    if lse is not None:
        l = lse.cpu().double()
        assert torch.equal(torch.isinf(l), torch.isinf(rl))
        fin = torch.isfinite(rl)
        assert ((l - rl).abs()[fin] <= (e + 2.0 ** -20 * (1 + rl.abs()))[fin]).all()
    if m is not None:
        dm = (m.cpu().double() - rm).abs()
        assert (dm <= em + 2.0 ** -18 * (1 + rm.abs())).all(), dm.max()
    return out, lse, m


def _filled(B, H, T, D, max_pos=None, seed=0, outliers=True):
    c = Cache(B, H, max_pos or (T + 63) // 64 * 64, D)
    k, v = _rand((B, T, H, D), 2 * seed + 1, outliers=outliers).cuda(), _rand((B, T, H, D), 2 * seed + 2).cuda()
    _append(c, k, v, _dev([0] * B))
    return c


# ------------------------------------------------------------------ rows ---

@pytest.mark.parametrize("B,H,S,D,start", [(1, 1, 1, 128, 0), (3, 2, 5, 128, 11), (2, 3, 37, 64, 0), (1, 8, 300, 128, 17),
                                           (4, 1, 33, 64, 63)])
def test_append_and_read_match_the_format(B, H, S, D, start):
    torch = _torch()
    c = Cache(B, H, 384, D)
    before = c.bits()
    k, v = _rand((B, S, H, D), 5, outliers=True), _rand((B, S, H, D), 6, 0.01)
    k[0, 0, 0, :64] = 1.25           # scale 0
    v[0, S - 1, 0, :] = 0.0
    k[0, S // 2, 0, :64] = torch.linspace(-1, 1, 64).bfloat16()
    v[0, S // 2, 0, 3] = 3.0e38      # max - min past the fp32 range
    v[0, S // 2, 0, 4] = -3.0e38
    lens = [start + 3 * b for b in range(B)]
    _append(c, k.cuda(), v.cuda(), _dev(lens))
    ko, vo = torch.full((B, S, H, D), 7.0, dtype=torch.bfloat16, device="cuda"), torch.empty(B, S, H, D,
                                                                                          dtype=torch.bfloat16, device="cuda")
    _api().kv4_read(c.h, ko.data_ptr(), vo.data_ptr(), S, _dev(lens).data_ptr())
    torch.cuda.synchronize()
    after = c.bits()
    for which, x, y in ((0, k, ko), (1, v, vo)):
        q, s, z = _quantize64(x.double().transpose(1, 2))
        word = (q.reshape(*q.shape[:-1], D // 8, 8) << torch.arange(0, 32, 4)).sum(-1)
        word = torch.where(word >= 2 ** 31, word - 2 ** 32, word).int()
        for b in range(B):
            rows = slice(lens[b], lens[b] + S)
            assert torch.equal(after[3 * which][b, :, rows], word[b])
            assert torch.equal(after[3 * which + 1][b, :, rows].view(torch.bfloat16).double(), s[b])
            assert torch.equal(after[3 * which + 2][b, :, rows].view(torch.bfloat16).double(), z[b])
            for t0, t1 in zip(before, after):  # every other row as it was
                assert torch.equal(t0[b, :, :lens[b]], t1[b, :, :lens[b]])
                assert torch.equal(t0[b, :, lens[b] + S:], t1[b, :, lens[b] + S:])
        ref = (q.double() * s.repeat_interleave(64, -1) + z.repeat_interleave(64, -1)).transpose(1, 2)
        d = (y.cpu().double() - ref).abs()
        assert (d <= (2.0 ** -8 + 2.0 ** -20) * ref.abs()).all()


def test_append_next_to_rounding_borders():
    """Quotients at exact halves go to the even neighbour; tiny offsets next to one decide it."""
    torch = _torch()
    c = Cache(1, 1, 64, 64)
    x = torch.zeros(1, 2, 1, 64)
    # scale 1, bias -4: the values -4 + n + 1/2 are exact halves
    x[0, 0, 0] = -4.0
    x[0, 0, 0, 1] = 11.0
    x[0, 0, 0, 2:17] = torch.arange(15) - 3.5
    # bias -4.5, scale 1: 0 is the half 4.5 (goes to 4); anything above 0 goes to 5, anything below to 4
    x[0, 1, 0] = -4.5
    x[0, 1, 0, 1] = 10.5
    x[0, 1, 0, 2] = 0.0
    x[0, 1, 0, 3] = 2.0 ** -30
    x[0, 1, 0, 4] = -(2.0 ** -30)
    x = x.bfloat16()
    _append(c, x.cuda(), x.cuda(), _dev([0]))
    torch.cuda.synchronize()
    q = ((c.t[0][0, 0, :2].cpu().long()[..., None] >> torch.arange(0, 32, 4)) & 15).reshape(2, 64)
    assert torch.equal(q, _quantize64(x[0, :, 0].double())[0])
    assert q[0, 2:17].tolist() == [0, 2, 2, 4, 4, 6, 6, 8, 8, 10, 10, 12, 12, 14, 14]
    assert q[1, 2:5].tolist() == [4, 5, 4]


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_append_of_a_non_finite_value_marks_its_group(bad):
    torch = _torch()
    c = Cache(1, 2, 64, 128)
    k = _rand((1, 3, 2, 128), 1)
    k[0, 1, 1, 70] = bad
    v = _rand((1, 3, 2, 128), 2)
    _append(c, k.cuda(), v.cuda(), _dev([4]))
    ko = torch.empty(1, 3, 2, 128, dtype=torch.bfloat16, device="cuda")
    _api().kv4_read(c.h, ko.data_ptr(), 0, 3, _dev([4]).data_ptr())
    torch.cuda.synchronize()
    nan = torch.isnan(ko.cpu())
    want = torch.zeros(1, 3, 2, 128, dtype=torch.bool)
    want[0, 1, 1, 64:] = True
    assert torch.equal(nan, want)


def test_append_strided_rows_of_a_fused_projection():
    """K and V as slices of one [B, S, (Hq + 2 Hkv) D] projection, and from an unaligned offset."""
    torch = _torch()
    B, S, H, D = 2, 9, 2, 128
    base = _rand((B, S, 10 * D + 8), 3).cuda()
    for shift in (0, 3):
        k = base[..., 4 * D + shift:6 * D + shift].unflatten(-1, (H, D))
        v = base[..., 6 * D + shift:8 * D + shift].unflatten(-1, (H, D))
        a, ref = Cache(B, H, 64, D), Cache(B, H, 64, D)
        _append(a, k, v, _dev([5, 0]))
        _append(ref, k.contiguous(), v.contiguous(), _dev([5, 0]), strides=False)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(a.bits(), ref.bits()))


def test_ragged_rows_and_the_end_of_the_cache():
    """Rows past n_new or past max_pos are not stored; the latter are reported."""
    torch = _torch()
    c = Cache(4, 2, 64, 64)
    before = c.bits()
    k = _rand((4, 6, 2, 64), 8).cuda()
    err = _dev([0])
    lens, n = _dev([0, 10, 20, 30]), _dev([6, 0, 3, -2])
    _append(c, k, k, lens, n, err=err)
    torch.cuda.synchronize()
    assert int(err) == 0
    after = c.bits()
    full = Cache(4, 2, 64, 64)
    _append(full, k, k, lens)
    torch.cuda.synchronize()
    full = full.bits()
    for t0, t1, tf in zip(before, after, full):
        for b, (p, m) in enumerate(zip([0, 10, 20, 30], [6, 0, 3, 0])):
            want = t0[b].clone()
            want[:, p:p + m] = tf[b, :, p:p + m]
            assert torch.equal(t1[b], want)
    _append(c, k, k, _dev([60, 64, 65, -1]), err=err)
    torch.cuda.synchronize()
    assert int(err) == 1
    y = torch.full((4, 6, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    lens, n = _dev([60, 64, 70, 0]), _dev([6, 6, 6, 2])
    _api().kv4_read(c.h, y.data_ptr(), 0, 6, lens.data_ptr(), n.data_ptr())
    torch.cuda.synchronize()
    z = (y.cpu() == 0).all(-1).all(-1)
    assert z.tolist()[0][4:] == [True, True] and not any(z.tolist()[0][:4])
    assert all(z.tolist()[1]) and all(z.tolist()[2]) and z.tolist()[3][2:] == [True] * 4


# ------------------------------------------------------------- attention ---

CASES = [
    # B, Hq, Hkv, D, S, total lengths
    (1, 1, 1, 128, 1, [1]),
    (1, 4, 1, 64, 1, [2]),
    (1, 16, 8, 128, 1, [519]),
    (3, 8, 2, 128, 1, [1, 64, 65]),
    (5, 14, 2, 64, 1, [15, 16, 17, 127, 128]),
    (2, 8, 1, 128, 1, [300, 33]),
    (2, 10, 2, 128, 1, [95, 97]),
    (1, 16, 1, 128, 1, [257]),
    (2, 32, 2, 64, 2, [100, 41]),
    (1, 8, 2, 128, 5, [812]),
    (2, 3, 3, 64, 3, [3, 31]),
    (2, 6, 2, 128, 8, [8, 200]),
    (1, 5, 1, 128, 7, [40]),
    (1, 4, 2, 128, 33, [33]),
    (1, 8, 2, 128, 64, [64]),
    (1, 8, 2, 64, 65, [190]),
    (2, 4, 1, 128, 130, [130, 331]),
    (1, 2, 1, 64, 257, [700]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("B,Hq,Hkv,D,S,total", CASES)
def test_attention(B, Hq, Hkv, D, S, total, causal):
    c = _filled(B, Hkv, max(total), D, seed=S)
    x = _rand((B, S, Hq, D), 77 + S, 1.5).cuda()
    _check_attention(c, x, _dev([t - S for t in total]), causal=causal, mass=True)


@pytest.mark.parametrize("S", [1, 4, 96])
def test_attention_ignores_what_lies_behind_the_lengths(S):
    """Rows past a sequence's length hold NaN scales; rows past n_new are padding."""
    torch = _torch()
    B, H, D, T = 5, 2, 128, 100
    c = Cache(B, H, 256, D)
    k = _rand((B, T + S, H, D), 1).cuda()
    lens, n = [0, T, 7, T, 50], [S, S, min(S, 2), 0, -3]
    for b in range(B):
        t = lens[b] + max(0, n[b])
        only = _dev([t if i == b else 0 for i in range(B)])
        _append(c, k, k, _dev([0] * B), only)
    x = _rand((B, S, 4, D), 4).cuda()
    out, lse, m = _check_attention(c, x, _dev(lens), _dev(n), mass=True)
    o, l = out.cpu(), lse.cpu()
    for b in range(B):
        rows = max(0, n[b])
        assert (o[b, rows:] == 0).all() and (l[b, rows:] == -float("inf")).all()
        assert torch.isfinite(l[b, :rows]).all()
    for causal in (True, False):
        out, lse, _ = _check_attention(c, x, _dev([0] * B), _dev([0] * B), causal=causal, mass=True)
        assert (out == 0).all()


@pytest.mark.parametrize("S,G", [(1, 4), (6, 4), (80, 2)])
def test_attention_at_the_end_of_the_cache(S, G):
    """Lengths that pass max_pos are cut there and reported."""
    c = _filled(2, 2, 128, 128, max_pos=128)
    x = _rand((2, S, 2 * G, 128), 5).cuda()
    err = _dev([0])
    _check_attention(c, x, _dev([128 - S, 3]), err=err, mass=True)
    assert int(err) == 0
    _check_attention(c, x, _dev([128 - S + 1, 128]), err=err)
    assert int(err) == 1


@pytest.mark.parametrize("S", [1, 3, 70])
def test_attention_strides(S):
    """q as a slice of a fused projection, out as a slice of a wider buffer; the rest of it is left alone."""
    torch = _torch()
    B, Hq, H, D, T = 2, 6, 2, 128, 150
    c = _filled(B, H, T, D)
    x = _rand((B, S, Hq * D + 2 * H * D), 9).cuda()[..., :Hq * D].unflatten(-1, (Hq, D))
    wide = torch.full((B, S, Hq + 1, 2 * D), 3.0, dtype=torch.bfloat16, device="cuda")
    out = wide[:, :, 1:, D:]
    got, _, _ = _check_attention(c, x, _dev([T - S, 40]), out=out)
    assert (wide[:, :, 0] == 3).all() and (wide[..., :D] == 3).all()
    ref, _ = _attend(c, x.contiguous(), _dev([T - S, 40]))
    assert torch.equal(ref, got)
    one = x[:1, :, :1].expand(B, S, Hq, D)  # broadcast queries
    _check_attention(c, one, _dev([T - S, 40]))


@pytest.mark.parametrize("S", [1, 48])
@pytest.mark.parametrize("kmul,vmul,qmul", [(1e-4, 1e-6, 30.0), (300.0, 3e4, 0.01), (1e6, 1e30, 1e-6),
                                            (1e-12, 1e-30, 1e12), (1.0, 1e-30, 1e-30)])
def test_attention_over_wide_ranges(S, kmul, vmul, qmul):
    """Keys, values and queries far outside the fp16 range."""
    c = Cache(1, 2, 192, 128)
    k = (_rand((1, 190, 2, 128), 3, outliers=True).float() * kmul).bfloat16().cuda()
    v = (_rand((1, 190, 2, 128), 4).float() * vmul).bfloat16()
    v[0, 50] = (v[0, 50].float() * 1e3).bfloat16()
    _append(c, k, v.cuda(), _dev([0]))
    x = (_rand((1, S, 8, 128), 6).float() * qmul).bfloat16().cuda()
    _check_attention(c, x, _dev([190 - S]), mass=True)


@pytest.mark.parametrize("S", [1, 40])
def test_attention_scale_signs_and_peaks(S):
    c = _filled(2, 2, 333, 64)
    x = _rand((2, S, 4, 64), 6).cuda()
    for scale in (0.0, -0.3, 4.0):
        _check_attention(c, x, _dev([333 - S, 20]), scale=scale, mass=True)


@pytest.mark.parametrize("S", [1, 40])
def test_attention_passes_on_a_nan_it_sees(S):
    """A NaN row makes the rows that see it NaN, and no others."""
    torch = _torch()
    c = Cache(2, 1, 128, 128)
    k = _rand((2, 100, 1, 128), 3)
    k[0, 99] = float("nan")
    _append(c, k.cuda(), k.cuda(), _dev([0, 0]))
    x = _rand((2, S, 2, 128), 4).cuda()
    out, _ = _attend(c, x, _dev([100 - S, 100 - S]))
    nan = torch.isnan(out.cpu()).all(-1).all(-1)
    assert nan[0].tolist() == [False] * (S - 1) + [True] and not nan[1].any()


def test_attention_without_lse_and_with_mass_only():
    torch = _torch()
    c = _filled(2, 2, 90, 128)
    x = _rand((2, 2, 8, 128), 1).cuda()
    a, _, ma = _check_attention(c, x, _dev([88, 30]), mass=True, want_lse=False)
    b, _, mb = _check_attention(c, x, _dev([88, 30]), mass=True)
    assert torch.equal(a, b) and torch.equal(ma, mb)


@pytest.mark.parametrize("S,G,T", [(1, 4, 3000), (5, 4, 700), (128, 2, 900)])
def test_attention_is_repeatable(S, G, T):
    """The same call gives the same bits, whatever the scratch held."""
    torch = _torch()
    c = _filled(3, 2, T, 128)
    x = _rand((3, S, 2 * G, 128), 1).cuda()
    lens = _dev([T - S, T // 2, 10])
    m = [torch.zeros(3, 2, c.max_pos, device="cuda") for _ in range(2)]
    n = max(16, _api().kv4_attention_scratch_bytes(c.h, S, 2 * G))
    one, l1 = _attend(c, x, lens, mass=m[0])
    two, l2 = _attend(c, x, lens, mass=m[1], scratch=torch.zeros(n, dtype=torch.uint8, device="cuda"))
    assert torch.equal(one, two) and torch.equal(l1, l2) and torch.equal(*m)


def _long(S, Hq, Hkv, T, B, D):
    """A ragged call against a 64-bit computation on the GPU."""
    torch = _torch()
    c = _filled(B, Hkv, T, D)
    g = np.random.default_rng(T)
    total = [T] + [int(t) for t in g.integers(S, T + 1, B - 1)]
    x = _rand((B, S, Hq, D), 12, 1.5).cuda()
    m = torch.zeros(B, Hkv, c.max_pos, device="cuda")
    out, lse = _attend(c, x, _dev([t - S for t in total]), mass=m)
    K, V = c.values64(0).cuda(), c.values64(1).cuda()
    G = Hq // Hkv
    for b in range(B):
        t = total[b]
        for h in range(Hkv):
            qr = x[b, :, h * G:(h + 1) * G].double()
            k, v = K[b, h, :t], V[b, h, :t]
            s = torch.einsum("igd,jd->igj", qr, k) * D ** -0.5
            hide = torch.arange(t, device="cuda")[None, :] > torch.arange(t - S, t, device="cuda")[:, None]
            s = s.masked_fill(hide[:, None], -float("inf"))
            z = torch.logsumexp(s, -1)
            p = torch.exp(s - z[..., None])
            ref = torch.einsum("igj,jd->igd", p, v)
            e = (2.0 ** -11 + 2.0 ** -16) * D ** -0.5 * torch.einsum("igd,jd->igj", qr.abs(), k.abs()).amax(-1)
            tol = 3 * v.abs().max() * (2.0 ** -10 + torch.expm1(2 * e))[..., None] + 2.0 ** -8 * ref.abs()
            assert ((out[b, :, h * G:(h + 1) * G].double() - ref).abs() <= tol).all()
            assert ((lse[b, :, h * G:(h + 1) * G].double() - z).abs() <= e + 2.0 ** -20 * (1 + z.abs())).all()
            em = (p * torch.expm1(2 * e)[..., None]).sum((0, 1))
            pm = p.sum((0, 1))
            assert ((m[b, h, :t].double() - pm).abs() <= em + 2.0 ** -18 * (1 + pm)).all()
        assert (m[b, :, t:] == 0).all()


@pytest.mark.parametrize("S,Hq,Hkv,T,B", [(1, 32, 8, 20000, 1), (1, 8, 1, 9000, 2), (1, 16, 4, 700, 40),
                                          (16, 16, 1, 4000, 1), (300, 4, 1, 3000, 1)])
def test_attention_long(S, Hq, Hkv, T, B):
    """Lengths that are split over many thread blocks."""
    _long(S, Hq, Hkv, T, B, 128)


@pytest.mark.parametrize("S,Hq,Hkv,T,B,D", [(1, 16, 1, 9000, 2, 128), (5, 8, 2, 9001, 1, 128), (5, 8, 2, 5000, 3, 64),
                                            (1, 6, 1, 12345, 1, 64), (1, 64, 1, 3001, 2, 128), (130, 2, 1, 4111, 2, 64),
                                            (40, 8, 2, 2500, 3, 128), (700, 2, 1, 701, 1, 128)])
def test_attention_long_forms(S, Hq, Hkv, T, B, D):
    """More columns per kv head and both head sizes, where the keys are split."""
    _long(S, Hq, Hkv, T, B, D)


def test_attention_of_many_sequences_in_a_long_cache():
    """More sequences than a warp plans for, many of them empty, some without new rows."""
    torch = _torch()
    B, H, D, T = 150, 1, 64, 2048
    c = Cache(B, H, T, D)
    g = np.random.default_rng(5)
    total = g.integers(1, 300, B)
    total[::7] = 0
    total[3] = 2048
    n = np.where(total > 0, 1, 0)
    k = _rand((B, 2048, H, D), 1).cuda()
    _append(c, k, k, _dev([0] * B), _dev(total))
    x = _rand((B, 1, 4, D), 2).cuda()
    seq, new = _dev(total - n), _dev(n)
    err = _dev([0])
    _check_attention(c, x, seq, new, mass=True, err=err)
    assert int(err) == 0


@pytest.mark.parametrize("S,Hq", [(96, 4), (200, 2), (7, 4)])
def test_attention_padded_batch_in_a_long_cache(S, Hq):
    """Rows past n_new and empty sequences where the keys are split over thread blocks; padding queries are NaN."""
    torch = _torch()
    B, H, D, T = 4, 2, 128, 6000
    c = Cache(B, H, 6400, D)
    k = _rand((B, T, H, D), 1).cuda()
    lens, n = [5000, 0, 0, 17], [S, 3, 0, S // 2]
    for b in range(B):
        t = lens[b] + n[b]
        _append(c, k, k, _dev([0] * B), _dev([t if i == b else 0 for i in range(B)]))
    x = _rand((B, S, Hq, D), 4)
    for b in range(B):
        x[b, n[b]:] = float("nan")
    out, lse = _attend(c, x.cuda(), _dev(lens), _dev(n))
    ref = _attend(c, torch.nan_to_num(x).cuda(), _dev(lens), _dev(n))
    assert torch.equal(out, ref[0]) and torch.equal(lse, ref[1])
    for b in range(B):
        assert (out[b, n[b]:] == 0).all() and (lse[b, n[b]:] == -float("inf")).all()
        assert torch.isfinite(out[b, :n[b]].float()).all()
    rows = [0, 1, 2, n[3] - 1]  # a few rows against the formula
    K, V = c.values64(0).cuda(), c.values64(1).cuda()
    for b in (0, 1, 3):
        for i in [r for r in rows if r < n[b]]:
            for h in range(Hq):
                kk, vv = K[b, h // (Hq // H), :lens[b] + i + 1], V[b, h // (Hq // H), :lens[b] + i + 1]
                s = (kk @ x[b, i, h].cuda().double()) * D ** -0.5
                p = torch.softmax(s, 0)
                e = (2.0 ** -11 + 2.0 ** -16) * D ** -0.5 * float((kk.abs() @ x[b, i, h].cuda().double().abs()).max())
                o = p @ vv
                tol = 3 * vv.abs().max() * (2.0 ** -10 + np.expm1(2 * e)) + 2.0 ** -8 * o.abs()
                assert ((out[b, i, h].double() - o).abs() <= tol).all()


@pytest.mark.parametrize("S,T", [(1, 700), (1, 9000), (90, 700)])
def test_attention_over_negative_scales(S, T):
    """A cache whose scales are negative (bias at the group's largest value), as another quantizer may leave it."""
    torch = _torch()
    a = _filled(1, 2, T, 128)
    b = Cache(1, 2, a.max_pos, 128)
    for w in (0, 3):  # q -> 15 - q, bias -> bias + 15 scale, scale -> -scale: exact where bias + 15 scale is a bf16
        s = a.t[w + 1].view(torch.bfloat16).float()
        b.t[w].copy_(~a.t[w])
        b.t[w + 1].copy_((-s).bfloat16().view(torch.int16))
        b.t[w + 2].copy_((a.t[w + 2].view(torch.bfloat16).float() + 15 * s).bfloat16().view(torch.int16))
    x = _rand((1, S, 4, 128), 3).cuda()
    out, lse = _attend(b, x, _dev([T - S]))
    K, V = b.values64(0)[0, :, :T].cuda(), b.values64(1)[0, :, :T].cuda()
    for h in range(4):
        s = torch.einsum("id,jd->ij", x[0, :, h].double(), K[h // 2]) * 128 ** -0.5
        s = s.masked_fill(torch.arange(T, device="cuda")[None] > torch.arange(T - S, T, device="cuda")[:, None], -float("inf"))
        p = torch.softmax(s, -1)
        o = p @ V[h // 2]
        e = (2.0 ** -11 + 2.0 ** -16) * 128 ** -0.5 * (x[0, :, h].double().abs() @ K[h // 2].abs().T).max()
        assert ((out[0, :, h].double() - o).abs() <= 3 * V.abs().max() * (2.0 ** -10 + torch.expm1(2 * e)) + 2.0 ** -8 * o.abs()).all()


def test_offsets_past_32_bits():
    """The last sequence of a cache whose words span more than 4 GiB."""
    torch, q = _torch(), _api()
    B, H, M, D = 65, 8, 131072, 128
    t = []
    for _ in range(2):
        t.append(torch.empty(B, H, M, D // 8, dtype=torch.int32, device="cuda"))
        t += [torch.empty(B, H, M, D // 64, dtype=torch.int16, device="cuda") for _ in range(2)]
    big = q.Kv4(*[x.data_ptr() for x in t], B, H, M, D)
    assert t[0].numel() * 4 > 1 << 32
    small = _filled(1, H, 70, D)
    lens, zero = [0] * B, [0] * B
    lens[-1], zero[-1] = M - 70, 70
    lens, zero = _dev(lens), _dev(zero)
    k, v = _rand((1, 70, H, D), 1, outliers=True).cuda(), _rand((1, 70, H, D), 2).cuda()
    q.kv4_append(big, k.expand(B, 70, H, D).data_ptr(), v.data_ptr(), 70, lens.data_ptr(), zero.data_ptr(),
                 k_strides=(0, H * D, D), v_strides=(0, H * D, D))
    for a, b in zip(t, small.t):
        assert torch.equal(a[-1, :, M - 70:], b[0, :, :70])
    # everything before the last rows: one repeated row of weight next to nothing
    for which in range(2):
        t[3 * which][-1] = 0
        t[3 * which + 1][-1] = 0
        t[3 * which + 2][-1] = 0
    q.kv4_append(big, k.data_ptr(), v.data_ptr(), 70, lens.data_ptr(), zero.data_ptr(),
                 k_strides=(0, H * D, D), v_strides=(0, H * D, D))
    x = _rand((1, 1, 8, D), 3).cuda()
    out = torch.empty(B, 1, 8, D, dtype=torch.bfloat16, device="cuda")
    lse = torch.empty(B, 1, 8, device="cuda")
    n = q.kv4_attention_scratch_bytes(big, 1, 8)
    scratch = torch.empty(n + 16, dtype=torch.uint8, device="cuda")
    seq = torch.zeros(B, dtype=torch.int32, device="cuda")
    seq[-1] = M - 1
    new = torch.zeros(B, dtype=torch.int32, device="cuda")
    new[-1] = 1
    mass = torch.zeros(B, H, M, device="cuda")
    q.kv4_attention(big, x.data_ptr(), out.data_ptr(), 1, 8, 0.1, seq.data_ptr(), scratch.data_ptr(), scratch.numel(),
                    n_new_ptr=new.data_ptr(), lse_ptr=lse.data_ptr(), mass_ptr=mass.data_ptr(), q_strides=(0, 0, D))
    K, V = small.values64(0)[0].cuda(), small.values64(1)[0].cuda()
    for h in range(8):
        s = 0.1 * (K[h, :70] @ x[0, 0, h].double())
        s = torch.cat([torch.zeros(M - 70, device="cuda").double(), s])
        p = torch.softmax(s, 0)
        ref = p[-70:] @ V[h, :70]
        assert ((out[-1, 0, h].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-2 * p[-70:].max() * V[h, :70].abs().max() * 70).all()
        assert abs(float(lse[-1, 0, h]) - float(torch.logsumexp(s, 0))) < 1e-3
        assert ((mass[-1, h].double() - p).abs() <= 1e-2 * p + 1e-9).all()
    assert (out[:-1] == 0).all() and (mass[:-1] == 0).all()


# -------------------------------------------------------------- eviction ---

def _evict(src, dst, ms, md, lens, new, keep, recent, index=None):
    torch, q = _torch(), _api()
    n = q.kv4_evict_scratch_bytes(src.h, keep)
    scratch = torch.full((n + 16,), 0xFF, dtype=torch.uint8, device="cuda")
    q.kv4_evict(src.h, dst.h, ms.data_ptr(), md.data_ptr(), lens.data_ptr(), new.data_ptr(), keep, recent,
                scratch.data_ptr(), n, index_ptr=0 if index is None else index.data_ptr(),
                stream=torch.cuda.current_stream().cuda_stream)


def _kept(mass, n, keep, recent):
    """Kept positions of one head: float64 weights, the lower position first among equals."""
    if n <= keep:
        return np.arange(n)
    old = n - recent
    m = np.where(np.isnan(mass[:old]), np.inf, mass[:old])
    order = sorted(range(old), key=lambda j: (not np.isnan(mass[j]), -m[j], j))
    return np.concatenate([np.sort(np.array(order[:keep - recent], dtype=np.int64)), np.arange(old, n)]).astype(np.int64)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("H,D,lens,keep,recent", [
    (1, 128, [1], 1, 0), (1, 64, [2], 1, 1), (2, 128, [0, 5, 30, 100], 30, 7), (3, 64, [700, 16, 512, 513], 512, 64),
    (2, 128, [2500, 1025, 1024, 3], 1024, 0), (1, 128, [5000], 4999, 4999), (2, 64, [4096, 4000], 1, 0),
    (8, 128, [3001], 2000, 333)])
def test_evict(H, D, lens, keep, recent, inplace):
    torch = _torch()
    B, T = len(lens), max(lens)
    src = _filled(B, H, T, D, seed=T)
    g = torch.Generator().manual_seed(T + keep)
    mass = torch.exp(2 * torch.randn(B, H, src.max_pos, generator=g))
    mass[torch.rand(mass.shape, generator=g) < 0.3] = 0.0   # ties
    mass[torch.rand(mass.shape, generator=g) < 0.1] = -0.0
    mass[torch.rand(mass.shape, generator=g) < 0.1] = 0.125
    mass[0, 0, T // 2] = float("nan")
    mass[-1, -1, T // 3] = float("inf")
    mass[-1, 0, 0] = -1.0
    dst = src if inplace else Cache(B, H, (keep + 15) // 16 * 16, D)
    s0, d0 = src.bits(), dst.bits()
    ms = mass.cuda()
    md = ms if inplace else torch.full((B, H, dst.max_pos), 9.0, device="cuda")
    md0 = md.cpu().clone()
    ln = _dev(lens)
    new = ln if inplace else _dev([-5] * B)
    index = _dev(np.full((B, H, keep), 77))
    _evict(src, dst, ms, md, ln, new, keep, recent, index)
    torch.cuda.synchronize()
    got = dst.bits()
    assert new.tolist() == [min(n, keep) for n in lens]
    for b, n in enumerate(lens):
        for h in range(H):
            ids = _kept(mass[b, h].double().numpy(), n, keep, recent)
            m = len(ids)
            assert index[b, h].tolist() == ids.tolist() + [-1] * (keep - m)
            for t0, t1, td in zip(s0, got, d0):
                assert torch.equal(t1[b, h, :m], t0[b, h, ids])
                if not inplace:
                    assert torch.equal(t1[b, h, m:], td[b, h, m:])
                elif n <= keep:
                    assert torch.equal(t1[b, h], t0[b, h])
                else:
                    assert torch.equal(t1[b, h, n:], t0[b, h, n:])
            a, w = md[b, h, :m].cpu(), mass[b, h, ids]
            assert torch.equal(torch.nan_to_num(a, nan=-7.0), torch.nan_to_num(w, nan=-7.0))
            if not inplace:
                assert torch.equal(md[b, h, m:].cpu(), md0[b, h, m:])
    if not inplace:
        assert all(torch.equal(x, y) for x, y in zip(src.bits(), s0))


@pytest.mark.parametrize("lens,cap,keep,recent", [([20000, 9000, 16384, 16385], 20480, 6000, 100), ([65000, 100, 33001], 65536, 4097, 0),
                                                 ([150001], 150016, 70000, 3), ([131072], 131072, 10, 10)])
def test_evict_positions_of_long_caches(lens, cap, keep, recent):
    """Lengths that take several thread blocks, or more positions than those hold; ties across their borders."""
    torch = _torch()
    B = len(lens)
    src, dst = Cache(B, 1, cap, 64), Cache(B, 1, (keep + 15) // 16 * 16, 64)
    g = np.random.default_rng(cap)
    m = np.exp(g.normal(size=(B, 1, cap))).astype(np.float32)
    m[g.random(m.shape) < 0.3] = 0.5  # the threshold falls among equals
    ms, md = torch.from_numpy(m).cuda(), torch.zeros(B, 1, dst.max_pos, device="cuda")
    for t in src.t:
        t.copy_(torch.arange(t[0, 0, :, 0].numel(), device="cuda").to(t.dtype)[None, None, :, None].expand_as(t))
    index, new = _dev(np.zeros((B, 1, keep))), _dev([0] * B)
    _evict(src, dst, ms, md, _dev(lens), new, keep, recent, index)
    assert new.tolist() == [min(n, keep) for n in lens]
    for b, n in enumerate(lens):
        order = np.lexsort((np.arange(n - recent), -m[b, 0, :n - recent]))[:keep - recent] if n > keep else np.arange(n)
        ids = np.concatenate([np.sort(order), np.arange(n - recent, n)]) if n > keep else order
        assert index[b, 0, :len(ids)].cpu().numpy().tolist() == ids.tolist() and (index[b, 0, len(ids):] == -1).all()
        at = torch.from_numpy(ids).cuda()
        assert torch.equal(md[b, 0, :len(ids)], ms[b, 0, at])
        assert all(torch.equal(d[b, 0, :len(ids)], t[b, 0, at]) for d, t in zip(dst.t, src.t))


def test_evict_all_equal_weights_keeps_the_lowest_positions():
    torch = _torch()
    src = _filled(1, 1, 300, 64)
    dst = Cache(1, 1, 64, 64)
    ms, md = torch.full((1, 1, src.max_pos), 2.0, device="cuda"), torch.zeros(1, 1, 64, device="cuda")
    index, new = _dev(np.zeros((1, 1, 50))), _dev([0])
    _evict(src, dst, ms, md, _dev([300]), new, 50, 10, index)
    assert index[0, 0].tolist() == list(range(40)) + list(range(290, 300))


# -------------------------------------------------------------- together ---

def _step(c, k, v, x, seq, mass, out, scratch):
    q = _api()
    stream = _torch().cuda.current_stream().cuda_stream
    q.kv4_append(c.h, k.data_ptr(), v.data_ptr(), k.shape[1], seq.data_ptr(), stream=stream)
    q.kv4_attention(c.h, x.data_ptr(), out.data_ptr(), x.shape[1], x.shape[2], 128 ** -0.5, seq.data_ptr(),
                    scratch.data_ptr(), scratch.numel(), mass_ptr=mass.data_ptr(), stream=stream)


def test_prompt_decode_and_eviction_together():
    """Prefill in two chunks, decode with accumulated weights, evict in place, decode on: every step
    against 64 bits on the cache's own contents, the same rows whether stored at once or in chunks."""
    torch = _torch()
    B, H, Hq, D, cap, keep, recent = 2, 2, 8, 128, 192, 96, 16
    c, whole = Cache(B, H, cap, D), Cache(B, H, cap, D)
    mass = torch.zeros(B, H, cap, device="cuda")
    seq = _dev([0, 0])
    k, v, x = [_rand((B, 150, n, D), i, outliers=i == 1).cuda() for i, n in ((1, H), (2, H), (3, Hq))]
    _append(whole, k, v, _dev([0, 0]))
    p = 0
    for n in (70, 33, 1, 1, 5):
        part = slice(p, p + n)
        _append(c, k[:, part], v[:, part], seq)
        before = mass.clone()
        out, lse, _ = _check_attention(c, x[:, part], seq)
        o2, _ = _attend(c, x[:, part], seq, mass=mass)
        assert torch.equal(out, o2)
        ref = _reference(c, x[:, part], seq.cpu(), None, True, D ** -0.5, before)
        assert ((mass.cpu().double() - ref[2]).abs() <= ref[3] + 2.0 ** -18 * (1 + ref[2].abs())).all()
        seq += n
        p += n
    assert all(torch.equal(a[:, :, :p], b[:, :, :p]) for a, b in zip(c.t, whole.t))
    # every row's weights sum to one: mass of a head = rows * query heads
    assert torch.allclose(mass[:, :, :p].sum(-1), torch.full((B, H), 110.0 * Hq / H, device="cuda"), rtol=1e-3)
    index = _dev(np.zeros((B, H, keep)))
    old = c.bits()
    mold = mass.cpu().double().numpy()
    _evict(c, c, mass, mass, seq, seq, keep, recent, index)
    assert seq.tolist() == [keep, keep]
    for b in range(B):
        for h in range(H):
            ids = _kept(mold[b, h], 110, keep, recent)
            assert index[b, h].tolist() == ids.tolist()
            assert all(torch.equal(n[b, h, :keep].cpu(), o[b, h, ids]) for n, o in zip(c.t, old))
    for n in (1, 3):
        part = slice(p, p + n)
        _append(c, k[:, part], v[:, part], seq)
        _check_attention(c, x[:, part], seq, mass=True)
        seq += n
        p += n


def test_captured_step_replays_at_every_length():
    """append + attention captured once, replayed while the device lengths advance, equals eager steps."""
    torch, q = _torch(), _api()
    B, H, Hq, D, cap = 2, 2, 8, 128, 256
    c, e = Cache(B, H, cap, D), Cache(B, H, cap, D)
    pre = _rand((B, 60, H, D), 1).cuda()
    for cc in (c, e):
        _append(cc, pre, pre, _dev([0, 0]))
    k, v, x = [torch.empty(B, 1, n, D, dtype=torch.bfloat16, device="cuda") for n in (H, H, Hq)]
    out = torch.empty(B, 1, Hq, D, dtype=torch.bfloat16, device="cuda")
    seq = _dev([60, 25])
    mass, me = torch.zeros(B, H, cap, device="cuda"), torch.zeros(B, H, cap, device="cuda")
    n = max(16, q.kv4_attention_scratch_bytes(c.h, 1, Hq))
    scratch = torch.empty(n, dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _step(c, k, v, x, seq, mass, out, scratch)
        seq += 1
    seq_e = _dev([60, 25])
    scratch_e = torch.empty(n, dtype=torch.uint8, device="cuda")
    out_e = torch.empty_like(out)
    for i in range(70):
        k.copy_(_rand((B, 1, H, D), 10 + i))
        v.copy_(_rand((B, 1, H, D), 500 + i))
        x.copy_(_rand((B, 1, Hq, D), 900 + i))
        g.replay()
        _step(e, k, v, x, seq_e, me, out_e, scratch_e)
        seq_e += 1
        assert torch.equal(out, out_e) and torch.equal(mass, me), i
    assert torch.equal(seq, seq_e)


def test_other_stream_and_two_calls_at_once():
    torch = _torch()
    c = _filled(2, 2, 900, 128)
    xs = [_rand((2, 1, 8, 128), 20 + i).cuda() for i in range(2)]
    lens = _dev([899, 500])
    want = [_attend(c, x, lens)[0].clone() for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(_attend(c, x, lens)[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,Hq,Hkv", [(1, 1, 1), (1, 6, 2), (5, 1, 1), (7, 2, 2), (2, 8, 2), (3, 3, 1), (15, 1, 1), (4, 4, 1),
                                      (17, 1, 1), (5, 16, 2), (63, 1, 1), (16, 4, 1), (13, 5, 1), (127, 1, 1), (32, 8, 2),
                                      (43, 3, 1), (51, 5, 1), (86, 3, 1)])
def test_weights_at_every_number_of_columns(S, Hq, Hkv, D):
    """1 to 258 columns per kv head: scores kept, recomputed and from kept queries; one sequence without rows, one that
    ends inside a tile, one whose queries past its rows are NaN."""
    torch = _torch()
    c = Cache(3, Hkv, 608, D)
    total = [601, 0, 258 + S]
    k = _rand((3, 601, Hkv, D), 1, outliers=True).cuda()
    _append(c, k, _rand((3, 601, Hkv, D), 2).cuda(), _dev([0, 0, 0]), _dev(total))
    n = [S, 0, (S + 1) // 2]
    x = _rand((3, S, Hq, D), 3)
    lens, new = _dev([t - r for t, r in zip(total, n)]), _dev(n)
    for causal in (True, False):
        _check_attention(c, x.cuda(), lens, new, causal=causal, mass=True)
    m = [torch.zeros(3, Hkv, c.max_pos, device="cuda") for _ in range(2)]
    _attend(c, x.cuda(), lens, new, mass=m[0])
    x[1] = x[2, n[2]:] = float("nan")
    _attend(c, x.cuda(), lens, new, mass=m[1])
    assert torch.equal(m[0], m[1]) and (m[0][1] == 0).all() and (m[0][2, :, total[2]:] == 0).all()


INF = float("inf")


@pytest.mark.parametrize("array,bad", [(1, INF), (1, -INF), (1, 3.0e38), (2, INF), (2, -INF), (4, INF), (4, -INF), (4, 3.0e38), (5, INF),
                                       (5, -INF)])  # scale and bias of K, of V
@pytest.mark.parametrize("S", [3, 20, 90])
def test_rows_before_an_infinity(S, array, bad):
    """Scales and biases of infinity (or past the range times 15) in a key that the last row alone sees: the other rows
    are those of a cache without it."""
    torch = _torch()
    a, b = _filled(1, 1, 300, 64), _filled(1, 1, 300, 64)
    b.t[array][0, 0, 299, 0] = int(torch.tensor(bad).bfloat16().view(torch.int16))
    x = _rand((1, S, 2, 64), 3).cuda()
    ma, mb = (torch.zeros(1, 1, a.max_pos, device="cuda") for _ in range(2))
    want, lse = _attend(a, x[:, :S - 1].contiguous(), _dev([300 - S]), mass=ma)
    got, lse_b = _attend(b, x, _dev([300 - S]), mass=mb)
    vm = a.values64(1)[0, 0, :300].abs().max().item()
    d = (got[:, :S - 1].double() - want.double()).abs()
    assert (d <= 2.0 ** -7 * want.double().abs() + 2.0 ** -9 * vm).all()
    assert ((lse_b[:, :S - 1] - lse).abs() <= 2.0 ** -16 * (1 + lse.abs())).all()


@pytest.mark.parametrize("S", [1, 8, 20, 64, 130])
def test_weights_beside_a_nan(S):
    """A NaN key makes the weights of the keys that its rows see NaN, and leaves those of other sequences and heads."""
    torch = _torch()
    c = Cache(2, 2, 320, 64)
    k = _rand((2, 300, 2, 64), 1)
    k[0, 299, 1] = float("nan")  # seen by the last row alone
    _append(c, k.cuda(), _rand((2, 300, 2, 64), 2).cuda(), _dev([0, 0]))
    x = _rand((2, S, 2, 64), 3).cuda()
    m = torch.zeros(2, 2, c.max_pos, device="cuda")
    out, _ = _attend(c, x, _dev([300 - S] * 2), mass=m)
    assert torch.isnan(m[0, 1, :300]).all() and (m[0, 1, 300:] == 0).all()
    assert torch.isfinite(m[1]).all() and torch.isfinite(m[0, 0]).all()
    assert torch.isfinite(out[0, :S - 1].float()).all() and torch.isfinite(out[1].float()).all()


@pytest.mark.parametrize("S,T", [(1, 300), (1, 9000), (90, 700), (90, 9000)])
def test_attention_in_place(S, T):
    torch, q = _torch(), _api()
    c = _filled(1, 2, T, 128)
    x = _rand((1, S, 8, 128), 3).cuda()
    lens = _dev([T - S])
    want = _attend(c, x, lens)[0]
    n = q.kv4_attention_scratch_bytes(c.h, S, 8)
    scratch = torch.empty(n, dtype=torch.uint8, device="cuda")
    q.kv4_attention(c.h, x.data_ptr(), x.data_ptr(), S, 8, 128 ** -0.5, lens.data_ptr(), scratch.data_ptr(), n,
                    stream=torch.cuda.current_stream().cuda_stream)
    assert torch.equal(x, want)


@pytest.mark.parametrize("S,Hq,T,D", [(1, 8, 9000, 128), (6, 8, 700, 64), (90, 4, 3000, 64), (90, 4, 700, 128)])
def test_weights_captured_and_beside_each_other(S, Hq, T, D):
    """A captured call replayed, and two calls on two streams with a scratch each, give what one call gives."""
    torch, q = _torch(), _api()
    c = _filled(2, 2, T, D)
    lens = _dev([T - S, T // 2])
    xs = [_rand((2, S, Hq, D), i).cuda() for i in (3, 4)]
    want = []
    for x in xs:
        m = torch.zeros(2, 2, c.max_pos, device="cuda")
        want.append((_attend(c, x, lens, mass=m), m))
    n = q.kv4_attention_scratch_bytes(c.h, S, Hq)
    scratch = [torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda") for _ in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    ms = [torch.zeros(2, 2, c.max_pos, device="cuda") for _ in xs]
    outs = [torch.empty_like(x) for x in xs]
    torch.cuda.synchronize()
    for _ in range(4):
        for s, x, m, o, w in zip(streams, xs, ms, outs, scratch):
            with torch.cuda.stream(s):
                m.zero_()
                _attend(c, x, lens, mass=m, out=o, scratch=w)
    torch.cuda.synchronize()
    for ((o, _), m), got, gm in zip(want, outs, ms):
        assert torch.equal(o, got) and torch.equal(m, gm)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for x, m, o in zip(xs, ms, outs):
            _attend(c, x, lens, mass=m, out=o, scratch=scratch[0], want_lse=False)
    for m in ms:
        m.zero_()
    g.replay()
    g.replay()
    torch.cuda.synchronize()
    for ((o, _), m), got, gm in zip(want, outs, ms):
        assert torch.equal(o, got) and torch.equal(2 * m, gm)


def test_host_memory_and_short_scratch_are_refused():
    torch, q = _torch(), _api()
    c = _filled(1, 1, 20, 64)
    x = _rand((1, 1, 1, 64), 1).cuda()
    host = [t.cpu() for t in c.t]
    hc = q.Kv4(*[(t.data_ptr() + 15) // 16 * 16 for t in host], 1, 1, c.max_pos, 64)
    with pytest.raises(q.Error):
        q.kv4_attention_scratch_bytes(hc, 1, 1)
    with pytest.raises(q.Error):
        q.kv4_append(hc, x.data_ptr(), x.data_ptr(), 1, _dev([0]).data_ptr())
    n = q.kv4_attention_scratch_bytes(c.h, 1, 1)
    if n:
        with pytest.raises(q.Error, match="scratch"):
            q.kv4_attention(c.h, x.data_ptr(), x.data_ptr(), 1, 1, 1.0, _dev([19]).data_ptr(), x.data_ptr(), n - 1)
    assert torch.cuda.current_device() == 0
