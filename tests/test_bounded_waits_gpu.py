"""Waits of the prompt and paged-cache kernels that run out (NMOE_WAIT_TRIES, the number of tries): the
call ends, what it could not compute is NaN and never a number, and the next call is as always."""
import pytest
import torch

from operators_ref import gdn
from test_linear_attn_prefill_gpu import TOL, Prompt

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
