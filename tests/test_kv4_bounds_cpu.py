"""What the bounds of test_gpu_kv4_bounds.py let through: the operators' own roundings, and no share of the keys that is lost
or scaled wrongly, no output of zeros.  Mistakes are planted in a 64-bit computation on the CPU."""
import pytest
import torch

from test_gpu_kv4 import Cache, _quantize64, _rand
from test_gpu_kv4_bounds import NORM, _bounds, _parts


def _cache(T, D, seed=0):
    c = Cache(1, 1, (T + 15) // 16 * 16, D, device="cpu")
    for which in (0, 1):
        q, s, z = _quantize64(_rand((1, 1, T, D), 2 * seed + 1 + which).double())
        w = (q.reshape(1, 1, T, D // 8, 8) << torch.arange(0, 32, 4)).sum(-1)
        c.t[3 * which][:, :, :T] = torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()
        c.t[3 * which + 1][:, :, :T] = s.bfloat16().view(torch.int16)
        c.t[3 * which + 2][:, :, :T] = z.bfloat16().view(torch.int16)
    return c


def _rows_outside(c, x, T, out):
    """Share of the rows of `out` that the bounds of an element or of the norm refuse."""
    o, to, _, _, _, _ = _bounds(c, x, [T - x.shape[1]], [x.shape[1]])[0]
    d = (out - o).abs()
    return ((d > to).any(-1) | (d.norm(dim=-1) > NORM * o.norm(dim=-1))).double().mean().item()


@pytest.mark.parametrize("S,G,T,D", [(1, 8, 6000, 128), (5, 4, 3000, 64), (40, 1, 2000, 128)])
def test_lost_and_misjoined_shares_are_outside_the_bounds(S, G, T, D):
    c = _cache(T, D)
    x = _rand((1, S, G, D), 12, 1.5)
    right, _, z, tz, w, tw = _bounds(c, x, [T - S], [S])[0]
    assert _rows_outside(c, x, T, right) == 0
    assert _rows_outside(c, x, T, torch.zeros_like(right)) == 1
    for share in ((0, T // 16), (T // 2, T // 2 + T // 16), (T // 3, T // 3 + T // 32)):
        lost, _, zl, _, wl, _ = _bounds(c, x, [T - S], [S], leave_out=share)[0]
        assert _rows_outside(c, x, T, lost) == 1
        assert ((zl - z).abs() > tz).double().mean() > 0.9
        assert ((wl - w).abs() > tw)[:, share[0]:share[1]].double().mean() > 0.5
    # one share's values scaled by 1 + 1/8
    (k, _), (v, _) = _parts(c, 0), _parts(c, 1)
    s = D ** -0.5 * torch.einsum("igd,jd->igj", x[0].double(), k[0, 0, :T])
    s = s.masked_fill((torch.arange(T)[None] > torch.arange(T - S, T)[:, None])[:, None], -float("inf"))
    p = torch.softmax(s, -1)
    p[..., T // 4:T // 2] *= 1.125
    assert _rows_outside(c, x, T, torch.einsum("igj,jd->igd", p, v[0, 0, :T])) == 1


@pytest.mark.parametrize("S,G,T,D", [(1, 8, 6000, 128), (40, 1, 2000, 64)])
def test_the_operators_roundings_are_inside_the_bounds(S, G, T, D):
    """Probabilities and values rounded to fp16, the output to bf16."""
    c = _cache(T, D)
    x = _rand((1, S, G, D), 12, 1.5)
    (k, _), (v, _) = _parts(c, 0), _parts(c, 1)
    s = D ** -0.5 * torch.einsum("igd,jd->igj", x[0].double(), k[0, 0, :T])
    s = s.masked_fill((torch.arange(T)[None] > torch.arange(T - S, T)[:, None])[:, None], -float("inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.einsum("igj,jd->igd", (p * 128).half().double() / 128, v[0, 0, :T].half().double()) / p.sum(-1, keepdim=True)
    assert _rows_outside(c, x, T, o.bfloat16().double()) == 0
