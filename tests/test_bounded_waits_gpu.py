"""Waits of the prompt and paged-cache kernels that run out (NMOE_WAIT_TRIES, the number of tries): the
call ends, what it could not compute is NaN and never a number, and the next call is as always."""
import pytest
import torch

from operators_ref import Packed, gdn
from test_linear_attn_prefill_gpu import TOL, Prompt
from test_paged_attn_gpu import H, append, check_prefill, check_step, prefill, step

pytestmark = pytest.mark.gpu
FEW = [1, 10, 40, 100, 300]   # tries that may or may not be enough


def all_or_nan(got, ref, tol):
    """Heads of rows [..][heads][dim] that are NaN in full; the others are within tol of ref."""
    lost = torch.isnan(got).all(-1, keepdim=True)
    assert bool((lost | ((got.double() - ref).abs() <= tol)).all())
    return lost


@pytest.mark.parametrize("rows", [[200, 0, 70], [9001]])   # the second one in parts
@pytest.mark.parametrize("tries", [0] + FEW)
def test_linear_attn_prefill(monkeypatch, rows, tries):
    p = Prompt(rows, 1, 2, torch.float32, seed=31, spare=3)
    conv, delta = p.conv.double().clone(), p.delta.double().clone()
    ref = gdn(p.w, p.hk, p.hv, p.cu_host, p.qkv, p.z, p.alpha, p.beta, conv, delta)
    n = p.cu_host[-1]
    monkeypatch.setenv("NMOE_WAIT_TRIES", str(tries))
    out, c, d = p.run()
    torch.cuda.synchronize()
    monkeypatch.delenv("NMOE_WAIT_TRIES")
    lost = all_or_nan(out[:n].view(n, 2, 128), ref[:n].view(n, 2, 128), TOL * float(ref.abs().max()))
    gone = all_or_nan(d.flatten(2), delta.flatten(2), TOL * float(delta.abs().max()))
    assert torch.equal(c.double(), conv)
    assert bool((out[n:] == 7.0).all())
    if tries == 0:   # a copy takes longer than one look
        assert bool(lost.all()) and bool(gone[[b for b, r in enumerate(rows) if r]].all())
    assert torch.equal(d[[b for b, r in enumerate(rows) if not r]], p.delta[[b for b, r in enumerate(rows) if not r]])
    p.check(*p.run())


@pytest.mark.parametrize("page", [16, 64, 7])
@pytest.mark.parametrize("shape", [(16, 2, 256, 64), (6, 1, 128, 128)])
@pytest.mark.parametrize("tries", [0] + FEW)
def test_full_attn_prefill(monkeypatch, shape, page, tries):
    p = Packed([130, 0, 70, 300], [0, 5, 200, 900], page, *shape, seed=32, spare_rows=3, tail=float("nan"))
    append(p)
    ref, mass, reach = p.attention()
    monkeypatch.setenv("NMOE_WAIT_TRIES", str(tries))
    out = prefill(p)
    torch.cuda.synchronize()
    monkeypatch.delenv("NMOE_WAIT_TRIES")
    n = sum(p.rows)
    tol = H * ref.abs() + (H + 2 * H * reach) * mass + 1e-30   # as in check_prefill
    lost = all_or_nan(out.view(p.total, p.hq, p.d)[:n], ref[:n], tol[:n])
    assert bool((out[n:] == 7.0).all())
    if tries == 0:
        assert bool(lost.all())
    check_prefill(p, prefill(p))


@pytest.mark.parametrize("page", [16, 7])
@pytest.mark.parametrize("shape", [(16, 2, 256, 64), (6, 1, 128, 128)])
@pytest.mark.parametrize("tries", [0] + FEW)
def test_full_attn_step(monkeypatch, shape, page, tries):
    p = Packed([1] * 6, [0, 63, 5000, 64, 17, 1200], page, *shape, torch.float32, seed=33, tail=float("nan"))
    monkeypatch.setenv("NMOE_WAIT_TRIES", str(tries))
    out = step(p, torch.float32)
    torch.cuda.synchronize()
    monkeypatch.delenv("NMOE_WAIT_TRIES")
    again = step(p, torch.float32)   # appends what the first call may not have come to
    check_step(p, again)
    ref, mass, _ = p.attention()
    lost = all_or_nan(out.view(6, p.hq, p.d), ref, 2e-5 * mass.amax(-1, keepdim=True) + 1e-30)   # as in check_step
    if tries == 0:
        assert bool(lost.all())
