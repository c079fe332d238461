"""The prompt attention against a 64-bit statement of what its products read: queries scaled and rounded
to bf16. What is left between them, and so the tolerance, is small enough to show one wrong position:
  2^-8 of the value (the output is bf16) and 2^-8 of the sum of p |v| (p is), half a step each;
  where the fp32 arithmetic before the rounding of a query (2e-6 of the head's largest element, as for appended
  keys) may have gone to the neighbouring bf16 value, the score moves by that step times |k|, and the
  normalised weights by twice the largest such move."""
import math

import pytest
import torch

from operators_ref import Packed, prepared
from test_paged_attn_gpu import H, append, prefill

pytestmark = pytest.mark.gpu


def statement(p, scale=None):
    """(out, tolerance) of every packed row and head, float64."""
    out = torch.zeros(p.total, p.hq, p.d, dtype=torch.float64, device="cuda")
    tol = torch.full_like(out, 1e-30)
    by = (scale or p.d ** -0.5) / math.log(2)
    for b, n in enumerate(p.rows):
        r0, length = int(p.cu[b]), p.lens[b]
        if n == 0:
            continue
        pos = torch.arange(length - n, length, device="cuda")
        q = p.q[r0:r0 + n].reshape(n, p.hq, -1)
        x = prepared(q[..., :p.d], p.weights["q_norm"], pos, p.rotary) * by
        gate = torch.sigmoid(q[..., p.d:].double())
        off = 2e-6 * x.abs().amax(-1, keepdim=True)
        lo, hi = ((x + s * off).bfloat16().double() for s in (-1, 1))
        x = x.bfloat16().double()
        page, slot = p.places(b)
        k, v = p.k[page, slot].double(), p.v[page, slot].double()
        hidden = torch.arange(length, device="cuda")[None] > pos[:, None]
        for h in range(p.hq):
            kh = h // (p.hq // p.hk)
            w = torch.exp2((x[:, h] @ k[:, kh].T).masked_fill(hidden, -math.inf))
            w = w / w.sum(-1, keepdim=True)
            move = ((hi - lo)[:, h] @ k[:, kh].abs().T).masked_fill(hidden, 0).amax(-1, keepdim=True) * math.log(2)
            y, mass = w @ v[:, kh] * gate[:, h], w @ v[:, kh].abs() * gate[:, h]
            out[r0:r0 + n, h] = y
            tol[r0:r0 + n, h] += H * y.abs() + (H + 2 * move) * mass
    return out, tol


@pytest.mark.parametrize("shape", [(16, 2, 256, 64), (6, 1, 128, 128), (5, 1, 256, 256), (24, 4, 128, 64)])
@pytest.mark.parametrize("page,dtype", [(16, torch.bfloat16), (64, torch.float32), (48, torch.bfloat16), (7, torch.float32)])
def test_prefill(shape, page, dtype):
    p = Packed([1, 37, 300, 129], [5, 0, 0, 700], page, *shape, dtype, seed=81, tail=float("nan"))
    append(p)
    ref, tol = statement(p)
    got = prefill(p).double().view(p.total, p.hq, p.d)
    bad = ~((got - ref).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), torch.nonzero(bad)[:4].tolist(), float(((got - ref).abs() / tol).max()))


def test_a_position_too_many_would_show():
    """The tolerance at work, on the statement: each row without its first position is outside it nearly everywhere
    that the first position has weight."""
    p = Packed([64], [0], 16, 16, 2, 256, 64, seed=82)
    append(p)
    ref, tol = statement(p)
    page, slot = p.places(0)
    got = prefill(p).double().view(64, 16, 256)
    assert bool(((got - ref).abs() <= tol).all())
    out = torch.zeros_like(ref)
    pos = torch.arange(64, device="cuda")
    q = p.q.reshape(64, 16, -1)
    x = (prepared(q[..., :256], p.weights["q_norm"], pos, 64) / 16 / math.log(2)).bfloat16().double()
    k, v = p.k[page, slot].double(), p.v[page, slot].double()
    for h in range(16):
        s = (x[:, h] @ k[:, h // 8].T).masked_fill((pos[None] > pos[:, None]) | (pos[None] == 0), -math.inf)
        w = torch.exp2(s)
        out[:, h] = (w / w.sum(-1, keepdim=True).clamp(min=1e-300)) @ v[:, h // 8] * torch.sigmoid(q[:, h, 256:].double())
    assert float(((out - ref).abs() > tol)[1:16].double().mean()) > 0.5
